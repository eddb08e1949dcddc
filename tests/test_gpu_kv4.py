"""The 4-bit MLA cache on the GPU: packing and reading back bit for bit, attention against a plain
64-bit one with bounds derived from the roundings that the kernels make, refusals and odd calls.

Bounds of the attention, per element, for bf16 half steps h = 2^-8:
  scores   the products of bf16 numbers are exact in 32 bits; 576 of them are added in some order with
           at most 2^-23 lost per addition (tensor cores cut, they do not round), so a scaled score is
           off by ds <= 576 * 2^-23 * sum |scale q k|, and by 2^-22 of it for the scaling
  weights  exp(s - m): 2^-16 for the exponential and its argument (|s - m| <= 2^7 where it counts),
           2 ds for both scores; p is rounded to bf16 (h) before it multiplies v
  out      (h + 2 ds + 2^-16) * sum p |v|, plus h of the result for its own rounding and 2^-16 * sum p |v|
           for the sums in 32 bits
  lse      ds + 2^-16 + 2^-22 |lse|
  weights  per entry w * (2 h + 2 ds + 2^-16) for p and the result, and h * 2^-24 a head where p vanishes
"""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
H_BF16 = 2.0**-8


@pytest.fixture(scope="module")
def kv4():
    import asu_ascend_b200

    asu_ascend_b200.load()
    from asu_ascend_b200 import kv4

    return kv4


@pytest.fixture
def checked():
    """Every operator call synchronises and raises on a device status."""
    from asu_ascend_b200 import ops

    ops.set_status_checks(True)
    yield
    ops.set_status_checks(False)


def latents(n, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, 576, generator=g) * torch.exp(spread * torch.randn(1, 576, generator=g))
    return x


def random_pool(shape, seed):
    """Bytes of 4-bit rows with scales around 2^-6 .. 2^1 and finite rope values."""
    rng = np.random.default_rng(seed)
    b = rng.integers(0, 256, (*shape, O.ROW), dtype=np.uint8)
    b[..., :256] |= ((b[..., :256] & 0x0F) == 0) * np.uint8(8) | ((b[..., :256] & 0xF0) == 0) * np.uint8(0x80)
    b[..., 256:288] = rng.integers(12 * 8, 16 * 8, (*shape, 32), dtype=np.uint8)
    rope = torch.randn(*shape, 64, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
    b[..., 288:] = rope.view(torch.int16).numpy().view(np.uint8).reshape(*shape, 128)
    return b


# ---- rows --------------------------------------------------------------------------------------

@pytest.mark.parametrize("n,dtype,pad,offset,spread", [
    (1, torch.bfloat16, 0, 0, 1.0), (257, torch.bfloat16, 64, 0, 3.0), (33, torch.float16, 0, 0, 1.0),
    (40, torch.float16, 8, 0, 1.0), (19, torch.bfloat16, 3, 0, 2.0), (21, torch.float16, 8, 5, 1.0)])
def test_rows_match_the_oracle_byte_for_byte(kv4, checked, n, dtype, pad, offset, spread):
    x = latents(n, n, spread).clamp(-6e4, 6e4)
    x[0, :16] = 0.0                       # a group of zeros
    x[n // 2, 16:32] = torch.tensor([7.0, 0.5, 1.5, 2.5, -0.5, -1.5, 3.5, 6.5] * 2)  # scale 1: ties everywhere
    x[n // 2, 32:48] = 1e-7               # under the smallest scale
    buf = torch.zeros(n, 576 + pad + offset, dtype=dtype, device=DEV)
    src = buf[:, offset: offset + 576]
    src.copy_(x)
    slots = torch.randperm(2 * n + 3, generator=torch.Generator().manual_seed(1))[:n].to(torch.int32)
    if n > 4:
        slots[3] = -1
    pool = torch.full((2 * n + 3, 416), 0xA5, dtype=torch.uint8, device=DEV)
    kv4.pack_rows(src, pool, slots.to(DEV))
    want = np.full((2 * n + 3, 416), 0xA5, np.uint8)
    packed = O.pack(src.float().cpu().numpy())
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            want[s] = packed[i]
    assert np.array_equal(pool.cpu().numpy(), want)
    back = kv4.unpack_rows(pool, slots.to(DEV)).float().cpu().numpy()
    values = O.unpack(packed)
    values[slots.numpy() < 0] = 0.0
    assert np.array_equal(back.astype(np.float64), values)


def test_every_magnitude_and_every_tie_is_rounded_as_the_definition_says(kv4, checked):
    """Groups whose largest magnitude is each finite bf16 number in turn, and groups of all the ties of each scale:
    the division by 7, the scale's rounding and the quotients, byte for byte."""
    rng = np.random.default_rng(8)
    top = torch.arange(1 << 15, dtype=torch.int32)[:0x7F80].to(torch.int16).view(torch.bfloat16)  # 0 to the largest
    part = torch.from_numpy(rng.uniform(-1, 1, (top.numel(), 15)).astype(np.float32))
    groups = torch.cat([top[:, None], (top.float()[:, None] * part).to(torch.bfloat16)], 1)
    s = torch.from_numpy(O.scale_of(np.arange(256)).astype(np.float32))
    ties = s[:, None] * (torch.arange(-7, 7) + 0.5)[None]  # 2k + 1 times a number of four bits: exact
    ties = torch.cat([ties, 7 * s[:, None], -3 * s[:, None]], 1)
    assert torch.equal(ties.to(torch.bfloat16).float(), ties)
    groups = torch.cat([groups, ties.to(torch.bfloat16)])
    x = torch.zeros(groups.shape[0] // 32, 576, dtype=torch.bfloat16)
    x[:, :512] = groups.reshape(-1, 512)
    pool = kv4.new_pool(x.shape[0], device=DEV)
    kv4.pack_rows(x.to(DEV), pool)
    assert np.array_equal(pool.cpu().numpy(), O.pack(x.float().numpy()))


def test_every_code_and_scale_reads_back_exactly(kv4, checked):
    """256 rows, one per scale byte, with all nibbles."""
    b = np.zeros((256, 416), np.uint8)
    b[:, :256] = np.arange(256, dtype=np.uint8)[None]
    b[:, 256:288] = np.arange(256, dtype=np.uint8)[:, None]
    got = kv4.unpack_rows(torch.from_numpy(b).to(DEV)).float().cpu().numpy()
    assert np.array_equal(got.astype(np.float64), O.unpack(b))


def test_rows_in_order_in_a_wider_pool(kv4, checked):
    wide = torch.zeros(50, 448, dtype=torch.uint8, device=DEV)
    x = latents(17, 3).to(torch.bfloat16).to(DEV)
    kv4.pack_rows(x, wide[:, 16:432])
    want = O.pack(x.float().cpu().numpy())
    got = wide.cpu().numpy()
    assert np.array_equal(got[:17, 16:432], want) and not got[17:].any() and not got[:, :16].any()
    assert not got[:, 432:].any()
    assert np.array_equal(kv4.unpack_rows(wide[:, 16:432]).float().cpu().numpy()[:17].astype(np.float64), O.unpack(want))
    assert kv4.unpack_rows(wide[:, 16:432], torch.zeros(0, dtype=torch.int32, device=DEV)).shape == (0, 576)
    kv4.pack_rows(x[:0], wide[:, 16:432])


def test_rows_that_cannot_be_stored_are_reported(kv4):
    from asu_ascend_b200 import ops

    x = latents(6, 5).to(torch.bfloat16)
    x[1, 40], x[2, 17], x[3, 100] = float("nan"), float("inf"), float("-inf")
    pool = torch.zeros(6, 416, dtype=torch.uint8, device=DEV)
    kv4.pack_rows(x.to(DEV), pool)
    v = O.unpack(pool.cpu().numpy())
    fine = x.float().numpy().copy()
    fine[1, 40] = 0.0
    assert np.array_equal(v[[0, 1, 4, 5]], O.unpack(O.pack(fine[[0, 1, 4, 5]])))
    top = 7 * 15 / 8 * 2.0**13
    assert v[2, 17] == top and v[3, 100] == -top
    ops.set_status_checks(True)
    try:
        with pytest.raises(RuntimeError, match="BAD_SOURCE"):
            kv4.pack_rows(x.to(DEV), pool)
        with pytest.raises(RuntimeError, match="BAD_QUERY"):
            kv4.pack_rows(x[:1].to(DEV), pool, torch.tensor([6], dtype=torch.int32, device=DEV))
        with pytest.raises(RuntimeError, match="BAD_QUERY"):
            kv4.unpack_rows(pool, torch.tensor([-2], dtype=torch.int32, device=DEV))
    finally:
        ops.set_status_checks(False)
    assert not kv4.unpack_rows(pool, torch.tensor([-2, 6], dtype=torch.int32, device=DEV)).any()


# ---- attention ---------------------------------------------------------------------------------

def check(q, pool, slots, scale, got, lost=0.0):
    """got against the oracle, token by token; q a CPU bf16 tensor, pool / slots numpy arrays; `lost`: what the
    outputs may be off by for weights below the range of the exponent, relative to the largest value."""
    out = got.out.float().cpu().numpy().astype(np.float64)
    lse = got.lse.cpu().numpy().astype(np.float64)
    w = None if got.weights is None else got.weights.float().cpu().numpy().astype(np.float64)
    for t in range(q.shape[0]):
        p = pool[t] if pool.ndim == 3 else pool
        o, l, ww, mag, smag = O.attention(q[t].float().numpy(), p, slots[t], scale)
        ds = (576 * 2.0**-23 + 2.0**-22) * smag
        lim = (H_BF16 + 2 * ds[:, None] + 2 * 2.0**-16) * mag
        lim += H_BF16 * (np.abs(o) + lim)
        if lost:
            lim += lost * np.abs(O.unpack(p)[:, :512]).max()
        worst = np.abs(out[t] - o) - lim
        assert (worst <= 0).all(), (t, np.argwhere(worst > 0)[:4], worst.max())
        if np.isinf(l).any():
            assert np.array_equal(lse[t], l)
        else:
            assert (np.abs(lse[t] - l) <= ds + 2.0**-16 + 2.0**-22 * np.abs(l)).all(), t
        if w is not None:
            lim = ww * (2 * H_BF16 + 2 * ds.max() + 2.0**-16) * (1 + 2.0**-7) + H_BF16 * 2.0**-24 * q.shape[1]
            assert (np.abs(w[t] - ww) <= lim).all(), t
            assert not w[t][(slots[t] < 0) | (slots[t] >= p.shape[0])].any()


def case(T, H, K, S, own, seed, valid=1.0, loud=1.0):
    rng = np.random.default_rng(seed)
    pool = random_pool((T, S) if own else (S,), seed)
    slots = np.stack([rng.permutation(S)[:K] if K <= S else rng.integers(0, S, K) for _ in range(T)]).astype(np.int32)
    slots = slots.reshape(T, K)
    if valid < 1.0:
        slots[rng.random((T, K)) >= valid] = -1
    q = (torch.randn(T, H, 576, generator=torch.Generator().manual_seed(seed)) * loud).to(torch.bfloat16)
    return q, pool, slots


SHAPES = [  # tokens, heads, topk, pool rows, one pool per token, share of entries, size of q
    (1, 1, 1, 1, False, 1.0, 1.0),
    (1, 16, 100, 300, False, 1.0, 1.0),
    (2, 8, 31, 64, True, 0.7, 1.0),
    (3, 17, 65, 200, False, 1.0, 4.0),
    (1, 128, 2048, 4000, False, 1.0, 1.0),
    (5, 24, 777, 1000, True, 0.5, 1.0),
    (2, 33, 129, 150, True, 0.9, 2.0),
    (3, 64, 512, 700, False, 1.0, 1.0),
    (2, 65, 127, 300, True, 1.0, 1.0),
    (2, 100, 300, 500, True, 0.2, 1.0),
    (4, 128, 128, 200, True, 1.0, 0.1),
    (160, 16, 64, 100, False, 0.8, 1.0),
    (150, 128, 70, 100, False, 0.9, 1.0),
    (1, 5, 5000, 6000, False, 0.95, 1.0),
    (1, 70, 5000, 3000, False, 0.95, 3.0),
]


@pytest.mark.parametrize("T,H,K,S,own,valid,loud", SHAPES)
def test_attention_matches_the_oracle(kv4, checked, T, H, K, S, own, valid, loud):
    q, pool, slots = case(T, H, K, S, own, T * 1000 + H * 10 + K, valid, loud)
    got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 192.0**-0.5,
                            weights=True)
    check(q, pool, slots, 192.0**-0.5, got)
    bare = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 192.0**-0.5)
    assert bare.weights is None and torch.equal(bare.out, got.out) and torch.equal(bare.lse, got.lse)


@pytest.mark.parametrize("H", [16, 64, 128])
def test_tokens_without_entries_and_padding_in_every_place(kv4, checked, H):
    T, K, S = 9, 200, 256
    q, pool, slots = case(T, H, K, S, True, 77 + H)
    slots[0] = -1
    slots[1, 1:] = -1
    slots[2, :-1] = -1
    slots[3, :64] = -1
    slots[4, 64:] = -1
    slots[5, ::2] = -1
    slots[6, 130:140] = -1
    slots[8] = -1
    got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07, weights=True)
    check(q, pool, slots, 0.07, got)
    assert not got.out[0].any() and torch.isinf(got.lse[8]).all()
    none = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.empty(T, 0, dtype=torch.int32, device=DEV),
                             0.07, weights=True)
    assert not none.out.any() and (none.lse == -float("inf")).all() and none.weights.shape == (T, 0)


@pytest.mark.parametrize("H", [16, 96])
def test_rows_that_no_slot_names_do_not_matter(kv4, checked, H):
    """NaN and infinite rope parts in unnamed rows, and in row 0 next to padding."""
    T, K, S = 3, 150, 400
    q, pool, slots = case(T, H, K, S, True, 5, 0.8)
    for t in range(T):
        slots[t][slots[t] == 0] = -1
        named = set(slots[t].tolist())
        for r in range(S):
            if r not in named:
                pool[t, r, 288:] = np.tile(np.array([0xC0, 0x7F, 0x80, 0xFF], np.uint8), 32)  # NaN, -inf
    got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07, weights=True)
    check(q, pool, slots, 0.07, got)


@pytest.mark.parametrize("H", [3, 128])
def test_entries_named_twice_and_slots_outside_the_pool(kv4, H):
    T, K, S = 2, 90, 40
    q, pool, slots = case(T, H, K, S, False, 9)  # more entries than rows: repeats
    slots[1, 5], slots[1, 6], slots[0, 89] = S, -7, 2**31 - 1
    args = (q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07)
    check(q, pool, slots, 0.07, kv4.sparse_decode(*args, weights=True))
    from asu_ascend_b200 import ops

    ops.set_status_checks(True)
    try:
        with pytest.raises(RuntimeError, match="BAD_QUERY"):
            kv4.sparse_decode(*args)
    finally:
        ops.set_status_checks(False)


@pytest.mark.parametrize("H", [16, 128])
def test_large_scores_do_not_overflow(kv4, checked, H):
    """Scores of some thousands, of one sign each: the running maximum has to carry them."""
    T, K, S = 2, 300, 300
    q, pool, slots = case(T, H, K, S, False, 11)
    q = q * 60
    q[1] = q[1].abs()
    got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 1.0, weights=True)
    assert torch.isfinite(got.out.float()).all() and torch.isfinite(got.lse).all()
    check(q, pool, slots, 1.0, got)


@pytest.mark.parametrize("H,loud", [(16, 60.0), (24, 60.0), (64, 60.0), (128, 60.0), (16, 3.0), (64, 3.0), (128, 3.0)])
def test_scores_that_rise_from_tile_to_tile(kv4, checked, H, loud):
    """Enough tokens that one block walks several tiles of each, in the order of one head's scores, upwards or
    downwards: what was summed so far has to be scaled again and again, after tiles without any entry too."""
    T, K, S = 170, 500, 520
    q, pool, slots = case(T, H, K, S, False, 19, 0.97, loud)
    kv = O.unpack(pool)
    for t in range(T):
        s = kv[slots[t]] @ q[t, t % H].double().numpy()
        s[slots[t] < 0] = s.min()
        slots[t] = slots[t][np.argsort(s if t % 3 else -s)]
        if t % 5 == 0:
            slots[t, : 64 * (t % 4 + 1)] = -1
    got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 1.0, weights=True)
    # Scores this far apart leave outputs of 1e-30 where the large weights' values are 0 or cancel.  The
    # exponentials are relative to a score of the token, so their sum is at least 1; one below 2^-126 may count as 0,
    # and its bf16 form be off by half of the smallest step, 2^-134: K entries lose at most K (2^-126 + 2^-134) max|v|.
    # The output's own smallest step adds 2^-134, less than 2^-126 of the largest value.
    check(q, pool, slots, 1.0, got, K * 2.0**-125)


@pytest.mark.parametrize("H,qpad,qoff", [(16, 64, 0), (16, 0, 3), (128, 64, 0), (128, 8, 5), (40, 0, 1)])
def test_strided_operands(kv4, checked, H, qpad, qoff):
    """q as a slice of a wider projection (any alignment), pools in wider rows, slots as columns of a table."""
    T, K, S = 3, 140, 160
    q, pool, slots = case(T, H, K, S, True, 13)
    qb = torch.full((T, H, 576 + qpad + qoff), float("nan"), dtype=torch.bfloat16, device=DEV)
    qs = qb[:, :, qoff: qoff + 576]
    qs.copy_(q)
    wide = torch.full((T, S + 2, 448), 0xFF, dtype=torch.uint8, device=DEV)
    ps = wide[:, 1: S + 1, 16:432]
    ps.copy_(torch.from_numpy(pool))
    table = torch.full((T, K + 9), 2**30, dtype=torch.int32, device=DEV)
    ss = table[:, 4: K + 4]
    ss.copy_(torch.from_numpy(slots))
    got = kv4.sparse_decode(qs, ps, ss, 0.07, weights=True)
    check(q, pool, slots, 0.07, got)
    # heads and tokens swapped in memory
    qt = q.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    again = kv4.sparse_decode(qt, ps, ss, 0.07, weights=True)
    assert torch.equal(again.out, got.out) and torch.equal(again.weights, got.weights)


def test_slots_behind_four_gigabytes(kv4, checked):
    """Row offsets above 2^32 bytes: a pool of 10.4 million rows, the last of them named."""
    S = (1 << 32) // 416 + 100_000
    pool = torch.zeros(S, 416, dtype=torch.uint8, device=DEV)
    K = 64
    rows = random_pool((K,), 21)
    slots = torch.arange(S - K, S, dtype=torch.int32, device=DEV)
    pool[S - K:] = torch.from_numpy(rows).to(DEV)
    for H in (16, 128):
        q = torch.randn(1, H, 576, generator=torch.Generator().manual_seed(H)).to(torch.bfloat16)
        got = kv4.sparse_decode(q.to(DEV), pool, slots[None], 0.07, weights=True)
        check(q, rows, np.arange(K, dtype=np.int32)[None], 0.07, got)
    assert np.array_equal(kv4.unpack_rows(pool, slots).double().cpu().numpy(), O.unpack(rows))


@pytest.mark.parametrize("H", [16, 128])
def test_captured_calls_keep_their_own_workspaces(kv4, H):
    """Two graphs, replayed in turn and with eager calls in between, on new inputs; bit-equal to eager."""
    K, S = 700, 900
    graphs = []
    for T in (1, 3):
        q, pool, slots = case(T, H, K, S, False, 100 + T)
        dq, dp, ds = q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV)
        kv4.sparse_decode(dq, dp, ds, 0.07, weights=True)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = kv4.sparse_decode(dq, dp, ds, 0.07, weights=True)
        graphs.append((g, got, dq, dp, ds))
    for turn in range(3):
        for g, got, dq, dp, ds in graphs:
            dq.copy_(torch.randn(dq.shape, generator=torch.Generator().manual_seed(turn)))
            g.replay()
        for g, got, dq, dp, ds in graphs:
            want = kv4.sparse_decode(dq, dp, ds, 0.07, weights=True)
            for a, b in zip(got, want):
                assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(kv4):
    q, pool, slots = case(2, 128, 600, 900, False, 55)
    args = (q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07)
    want = kv4.sparse_decode(*args, weights=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            got.append(kv4.sparse_decode(*args, weights=True))
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


def test_four_bit_rows_through_the_managed_cache(kv4, checked):
    """sparse_mla.sparse_mla_decode over a paged cache of 4-bit rows: resolver, managed rows, attention."""
    from asu_ascend_b200 import sparse_mla

    bs, blocks, seq, H, K = 64, 20, 1200, 16, 256
    x = latents(blocks * bs, 8).to(torch.bfloat16).to(DEV)
    cache = kv4.new_pool(blocks, bs, device=DEV)
    kv4.pack_rows(x, cache.view(-1, 416))
    rng = np.random.default_rng(3)
    table = torch.from_numpy(rng.permutation(blocks).astype(np.int32)).to(DEV)
    mgr = sparse_mla.contexts_for_mla({"l": cache, "m": cache}, blocks * bs, bs, managed_slot_count=600, enabled=True,
                                      free_target=300)
    mgr.reset_single_request("r", seq, 1100, table)
    ctx = mgr.get_layer_context("l")
    flat = cache.view(-1, 416).cpu().numpy()
    for step in range(3):
        topk = rng.permutation(seq)[:K].astype(np.int32)
        topk[200:] = -1
        q = torch.randn(1, H, 576, generator=torch.Generator().manual_seed(step)).to(torch.bfloat16)
        out = sparse_mla.sparse_mla_decode(q.to(DEV), ctx, torch.from_numpy(topk)[None].to(DEV), table, cache, 0.07)
        at = np.where(topk >= 0, table.cpu().numpy()[topk // bs] * bs + topk % bs, -1).astype(np.int32)
        o, _, _, mag, smag = O.attention(q[0].float().numpy(), flat, at, 0.07)
        ds = (576 * 2.0**-23 + 2.0**-22) * smag
        lim = (H_BF16 + 2 * ds[:, None] + 2 * 2.0**-16) * mag
        assert (np.abs(out[0].float().cpu().numpy() - o) <= lim + H_BF16 * (np.abs(o) + lim)).all()


# ---- values that are not finite ----------------------------------------------------------------

def plant(q, pool, slots, shift):
    """NaN in a head's q, NaN in the rope part of a named row, an infinite value in a head's q, or nothing: by token."""
    for t in range(q.shape[0]):
        kind, h = (t + shift) % 4, (5 * t + shift) % q.shape[1]
        live = slots[t][slots[t] >= 0]
        if kind == 1:
            q[t, h, 7] = float("nan")
        elif kind == 2 and len(live):
            pool[t, live[len(live) // 2], 290:292] = (0xC0, 0x7F)
        elif kind == 3:
            q[t, h, 512 + 5] = float("inf")
            pool[t, :, 288 + 10: 288 + 12] = (0x80, 0x3F)  # times 1: an infinite score


@pytest.mark.parametrize("T,H,K", [
    (1, 16, 100), (1, 16, 700), (1, 64, 1500), (2, 33, 300), (37, 24, 777), (170, 16, 150), (150, 40, 260),
    (1, 128, 60), (1, 128, 700), (3, 100, 300), (150, 80, 130)])
def test_what_is_not_a_number_is_reported_as_such(kv4, checked, T, H, K):
    """A head whose scores are not numbers has NaN for out and lse, and the weights of the token's entries are NaN;
    entries that are not there keep weight 0, and other heads and tokens their values."""
    for shift in (1, 2, 3) if T == 1 else (0, 2):
        q, pool, slots = case(T, H, K, K + 50, True, 31 + T + H, 0.9)
        plant(q, pool, slots, shift)
        got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07,
                                weights=True)
        out, lse, w = (x.double().cpu().numpy() for x in got)
        seen = 0
        for t in range(T):
            with np.errstate(invalid="ignore"):
                o, l, ww, mag, smag = O.attention(q[t].float().numpy(), pool[t], slots[t], 0.07)
            bad = np.isnan(l)
            seen += bad.sum()
            assert np.array_equal(np.isnan(lse[t]), bad), t
            assert np.isnan(out[t][bad]).all(), t
            ds = (576 * 2.0**-23 + 2.0**-22) * smag
            lim = (H_BF16 + 2 * ds[:, None] + 2 * 2.0**-16) * mag
            lim += H_BF16 * (np.abs(o) + lim)
            assert (np.abs(out[t] - o) <= lim)[~bad].all(), t
            assert (np.abs(lse[t] - l) <= ds + 2.0**-16 + 2.0**-22 * np.abs(l))[~bad].all(), t
            assert not w[t][slots[t] < 0].any(), t
            assert np.array_equal(np.isnan(w[t]), np.isnan(ww)), t
            if not bad.any():
                lim = ww * (2 * H_BF16 + 2 * ds.max() + 2.0**-16) * (1 + 2.0**-7) + H_BF16 * 2.0**-24 * H
                assert (np.abs(w[t] - ww) <= lim).all(), t
        assert seen > 0


@pytest.mark.parametrize("T,H,K,split", [(1, 16, 300, 130), (3, 24, 777, 400), (170, 16, 300, 140), (2, 64, 260, 128),
                                         (1, 128, 300, 70), (80, 100, 300, 140)])
def test_scores_of_minus_infinity_add_nothing(kv4, checked, T, H, K, split):
    """The first entries' scores overflow to -inf (2^127 times -4), for whole tiles and more: they count as if they were
    not there, and a token that has no other entry gets what one without entries gets."""
    q, pool, slots = case(T, H, K, K + 9, True, 71 + H)
    q[:, :, 512] = 2.0**127
    want = slots.copy()
    for t in range(T):
        n = K if t % 3 == 2 else split
        pool[t, :, 288:290] = 0
        pool[t, slots[t, :n], 288:290] = (0x80, 0xC0)  # -4
        want[t, :n] = -1
    got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07, weights=True)
    check(q, pool, want, 0.07, got)


# ---- many tokens in a call ---------------------------------------------------------------------

@pytest.mark.parametrize("T,H,K,own,part", [(4100, 16, 2048, False, 2050), (1100, 64, 2048, False, 550),
                                            (700, 128, 2048, True, 350), (500, 128, 2048, False, 250)])
def test_weights_of_more_tokens_than_the_workspace_holds(kv4, checked, T, H, K, own, part):
    """Calls that are done in parts (256 MiB of softmax weights each): bit for bit the calls of those parts."""
    S = 300
    rng = np.random.default_rng(T)
    pool = random_pool((T, S) if own else (S,), 3)
    slots = rng.integers(-1, S, (T, K)).astype(np.int32)
    q = torch.randn(H, T, 576, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).transpose(0, 1)
    dq, dp = q.to(DEV), torch.from_numpy(pool).to(DEV)
    ds = torch.full((T, K + 5), -9, dtype=torch.int32, device=DEV)[:, 2: K + 2]
    ds.copy_(torch.from_numpy(slots))
    got = kv4.sparse_decode(dq, dp, ds, 0.07, weights=True)
    for t in range(0, T, part):
        at = slice(t, t + part)
        want = kv4.sparse_decode(dq[at], dp[at] if own else dp, ds[at], 0.07, weights=True)
        for a, b in zip(got, want):
            assert torch.equal(a[at], b)
    at = [0, 1, part - 1, part, part + 1, T - 1]
    some = kv4_of(got, at)
    check(q[at], pool[at] if own else pool, slots[at], 0.07, some)


def kv4_of(got, at):
    return type(got)(*(x[at] for x in got))


@pytest.mark.parametrize("T,H,K", [(65535, 1, 3), (5000, 20, 33), (3000, 70, 90)])
def test_many_tokens(kv4, checked, T, H, K):
    """A prompt's worth of tokens and the most that a call takes; a sample of them against the oracle."""
    S = 200
    rng = np.random.default_rng(T)
    pool = random_pool((S,), 4)
    slots = rng.integers(-1, S, (T, K)).astype(np.int32)
    q = torch.randn(T, H, 576, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16)
    got = kv4.sparse_decode(q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07, weights=True)
    assert not torch.isnan(got.out).any() and not torch.isnan(got.lse).any()
    at = np.unique(np.concatenate([[0, 1, T - 2, T - 1], rng.integers(0, T, 60)])).tolist()
    check(q[at], pool, slots[at], 0.07, kv4_of(got, at))


@pytest.mark.parametrize("T,H,K", [(60, 128, 300), (74, 80, 64), (148, 128, 130), (200, 100, 64), (148, 16, 300),
                                   (296, 40, 200)])
def test_tokens_of_a_cta_each_or_several(kv4, checked, T, H, K):
    """No token lies in several CTAs' ranges, so that the call has no pieces and, without weights, no workspace."""
    from asu_ascend_b200 import _lib

    assert _lib.lib.asu_kv4_attention_workspace_bytes(T, H, K, 0) == 0
    q, pool, slots = case(T, H, K, 400, False, 17 + T, 0.9)
    args = (q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07)
    got = kv4.sparse_decode(*args, weights=True)
    check(q, pool, slots, 0.07, got)
    bare = kv4.sparse_decode(*args)
    assert torch.equal(bare.out, got.out) and torch.equal(bare.lse, got.lse)


def test_pools_of_one_row_or_one_token_with_odd_strides(kv4, checked):
    """The strides of dimensions of one element do not reach the kernels."""
    one = torch.zeros(416, 1, dtype=torch.uint8, device=DEV).t()
    x = latents(1, 2).to(torch.bfloat16)
    kv4.pack_rows(x.to(DEV), one)
    want = O.pack(x.float().numpy())
    assert np.array_equal(one.cpu().numpy(), want)
    assert np.array_equal(kv4.unpack_rows(one).double().cpu().numpy(), O.unpack(want))
    odd = torch.zeros(1280, dtype=torch.uint8, device=DEV).as_strided((1, 1, 416), (425, 7, 1))
    odd.copy_(one[None])
    slots = np.array([[0, -1, 0]], np.int32)
    for H in (16, 128):
        q = torch.randn(1, H, 576, generator=torch.Generator().manual_seed(H)).to(torch.bfloat16)
        got = kv4.sparse_decode(q.to(DEV), odd, torch.from_numpy(slots).to(DEV), 0.07, weights=True)
        check(q, want, slots, 0.07, got)


# ---- several calls at once ---------------------------------------------------------------------

@pytest.mark.parametrize("shapes", [
    [(1, 16, 700), (2, 16, 600), (9, 16, 1000)],                 # clusters of 6, 5 and 8
    [(1, 16, 100), (2, 33, 300), (1, 64, 1024), (20, 24, 700)],  # of 1 (for the weights), 3, 8, 6
    [(61, 64, 300), (37, 24, 777), (170, 16, 150)],              # clusters of 2; without clusters
    [(2, 16, 600), (1, 128, 900), (37, 24, 777), (20, 40, 700), (80, 100, 130)]], ids=str)
def test_calls_of_several_kernels_on_several_streams(kv4, shapes):
    """Blocks that join in clusters, blocks that do not and the kernel for many heads, at the same time on the same SMs:
    bit for bit the results of one after the other."""
    calls = []
    for i, (T, H, K) in enumerate(shapes):
        q, pool, slots = case(T, H, K, K + 20, False, 300 + i, 0.95)
        args = (q.to(DEV), torch.from_numpy(pool).to(DEV), torch.from_numpy(slots).to(DEV), 0.07)
        calls.append((args, kv4.sparse_decode(*args, weights=True), kv4.sparse_decode(*args)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(40):
        i = turn * 3 % len(calls) if len(calls) % 3 else turn % len(calls)
        with torch.cuda.stream(streams[turn % 4]):
            got.append((i, kv4.sparse_decode(*calls[i][0], weights=turn % 5 != 0)))
    torch.cuda.synchronize()
    for i, g in got:
        args, full, bare = calls[i]
        for a, b in zip(g, full if g.weights is not None else bare):
            assert (a is None and b is None) or torch.equal(a, b)
