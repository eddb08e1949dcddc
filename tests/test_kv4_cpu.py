"""The 4-bit MLA cache and the attention-weight slot pools without a GPU: the row format's own
properties on the oracle, the refusals of the C entry points, of the torch operators and of the Python
objects, and the operators' shapes under torch's meta device."""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O


@pytest.fixture(scope="module")
def lib():
    from asu_ascend_b200 import _lib

    return _lib


# ---- the format --------------------------------------------------------------------------------

def test_values_are_exact_in_bf16_and_so_is_the_fused_form():
    """(n - 8) * s, and 136 * s of the one-fma form, need 8 significant bits at most."""
    s = O.scale_of(np.arange(256))
    v = (np.arange(16)[:, None] - 8.0) * s[None]
    assert np.array_equal(O.bf16_round(v.astype(np.float32)).astype(np.float64), v)
    assert np.array_equal(O.bf16_round((136.0 * s).astype(np.float32)).astype(np.float64), 136.0 * s)


def test_rounding_error_is_half_a_step():
    """s is a / 7 rounded by at most 1 part in 16, so |x| / s < 7.5 and no value is clamped: its error
    is at most s / 2 (one part in 2^20 spare for the division in the test)."""
    rng = np.random.default_rng(1)
    x = O.bf16_round((rng.standard_normal((40, 576)) * np.exp(2 * rng.standard_normal((40, 1)))).astype(np.float32))
    b = O.pack(x)
    back = O.unpack(b)
    s = np.repeat(O.scale_of(b[:, 256:288]), 16, 1)
    a = np.abs(x[:, :512].astype(np.float64)).reshape(40, 32, 16).max(2)
    assert (np.abs(O.scale_of(b[:, 256:288]) * 7 / a - 1) <= 1 / 16).all()
    assert (np.abs(back[:, :512] - x[:, :512]) <= s / 2 * (1 + 2.0**-20)).all()
    assert np.array_equal(back[:, 512:], x[:, 512:])


def test_scale_ties_go_to_the_even_byte():
    """a / 7 midway between two bytes' values is a number of 8 bits: 7 * (17..31 odd) / 16."""
    for odd in range(17, 32, 2):
        byte = O.nearest_scale(7.0 * odd / 16)
        below = (odd - 17) // 2 + 18 * 8
        assert byte == (below if below % 2 == 0 else below + 1)
    assert O.nearest_scale(0.0) == 0 and O.nearest_scale(1e30) == 255


def test_weight_pool_oracle_keeps_what_attention_reads():
    p = O.WeightPool(8, 2, 0.5)
    slot, hit, inst, ev = p.step([10, 11, 12, 13, 14, 15])
    assert slot == [0, 1, 2, 3, 4, 5] and not any(hit) and all(inst) and ev == []
    slot, hit, inst, ev = p.step([10, 20, 21, 20], slot, [0.1, 3.0, 0.2, 0.2, 2.0, 1.0])
    assert ev == [] and slot == [0, 6, 7, 6] and hit == [True, False, False, True]
    # nothing is free: two of the lowest leave; 12 and 13 tie at 0.1 with 10 lower but asked for
    slot, hit, inst, ev = p.step([10, 30], slot, [0.0, 0.0, 0.5, 0.0])
    assert ev == [12, 20] and slot == [0, 6]


# ---- C entry points ----------------------------------------------------------------------------

def test_pack_and_unpack_reject_before_launch(lib):
    L, A, G = lib.lib, lib.ASU_ERR_ARG, lib.ASU_ERR_ALIGN
    assert L.asu_kv4_pack(None, None, 0, 576, 0, None, None, 0, 416, None) == lib.ASU_OK
    assert L.asu_kv4_pack(None, None, 0, 576, 4, None, 16, 8, 416, None) == A
    assert L.asu_kv4_pack(None, 16, 0, 576, 4, None, None, 8, 416, None) == A
    assert L.asu_kv4_pack(None, 16, 2, 576, 4, None, 16, 8, 416, None) == A       # fp32 rows
    assert L.asu_kv4_pack(None, 16, 0, 576, 9, None, 16, 8, 416, None) == A       # more rows than the pool
    assert L.asu_kv4_pack(None, 16, 0, 576, -1, None, 16, 8, 416, None) == A
    assert L.asu_kv4_pack(None, 16, 0, 576, 4, None, 16, 8, 400, None) == A
    assert L.asu_kv4_pack(None, 16, 0, 576, 4, None, 8, 8, 416, None) == G
    assert L.asu_kv4_pack(None, 16, 0, 576, 4, None, 16, 8, 424, None) == G
    assert L.asu_kv4_pack(None, 17, 0, 576, 4, None, 16, 8, 416, None) == G
    assert L.asu_kv4_unpack(None, 16, 8, 416, None, 0, None, 576, None) == lib.ASU_OK
    assert L.asu_kv4_unpack(None, 16, 8, 416, None, 9, 16, 576, None) == A
    assert L.asu_kv4_unpack(None, 16, 8, 416, None, 4, 16, 575, None) == A
    assert L.asu_kv4_unpack(None, 16, 8, 416, None, 4, 16, 580, None) == G
    assert L.asu_kv4_unpack(None, 16, 8, 416, None, 4, 24, 576, None) == G


def _attention(L, **kw):
    a = dict(stream=None, q=16, qt=576, qh=576, pool=16, rows=8, pitch=416, pt=0, slots=16, st=4, tokens=1, heads=1,
             topk=4, scale=1.0, out=16, lse=16, weights=None, ws=16, size=1 << 40, status=None)
    a.update(kw)
    return L.asu_kv4_attention(*a.values())


def test_attention_rejects_before_launch(lib):
    L, A, G = lib.lib, lib.ASU_ERR_ARG, lib.ASU_ERR_ALIGN
    assert _attention(L, tokens=0) == lib.ASU_OK
    for bad in (dict(tokens=-1), dict(heads=129), dict(topk=16385), dict(tokens=65536), dict(q=None), dict(out=None),
                dict(lse=None), dict(slots=None), dict(pool=None), dict(scale=0.0), dict(scale=-1.0),
                dict(scale=float("inf")), dict(scale=float("nan")), dict(pitch=400), dict(rows=2**31),
                dict(qt=-1), dict(weights=16, ws=None), dict(weights=16, size=0)):
        assert _attention(L, **bad) == A, bad
    for bad in (dict(q=17), dict(pool=24), dict(pitch=424), dict(pt=8), dict(out=24), dict(lse=18), dict(ws=24)):
        assert _attention(L, **bad) == G, bad
    size = L.asu_kv4_attention_workspace_bytes
    assert size(1, 129, 4, 0) == -1 and size(-1, 1, 4, 0) == -1 and size(1, 1, 16385, 1) == -1
    assert size(0, 16, 2048, 0) >= 0


def test_attention_rejects_what_its_vector_stores_and_scaling_cannot_take(lib):
    L, A, G = lib.lib, lib.ASU_ERR_ARG, lib.ASU_ERR_ALIGN
    ok = dict(out=64, ws=64)
    for bad in (dict(out=48), dict(ws=48), dict(slots=18), dict(weights=17)):
        assert _attention(L, **(ok | bad)) == G, bad
    assert _attention(L, **ok, scale=3e38) == A  # times log2(e) it is infinite


def _step(L, **kw):
    a = dict(stream=None, t2s=16, s2t=16, score=16, stack=16, count=16, last=1 << 20, weight=16, wtype=2, n=4, decay=0.5,
             keep=None, query=16, slot=1 << 30, hit=16, inst=16, ev=16, ev_stride=4, evn=16, stats=None, status=None,
             R=1, K=100, S=8, Q=4, target=4)
    a.update(kw)
    return L.asu_weight_step(*a.values())


def test_weight_step_rejects_before_launch(lib):
    L, A = lib.lib, lib.ASU_ERR_ARG
    assert _step(L, R=0) == lib.ASU_OK
    for bad in (dict(t2s=None), dict(score=None), dict(count=None), dict(query=None), dict(slot=None), dict(evn=None),
                dict(S=16385), dict(Q=4097), dict(n=4097), dict(K=0), dict(S=0), dict(decay=-0.1), dict(decay=1.5),
                dict(decay=float("nan")), dict(wtype=1), dict(weight=None), dict(last=None), dict(ev_stride=3),
                dict(ev=None),
                # the new slots may overwrite the last ones row for row, not across rows
                dict(slot=1 << 20, n=3), dict(slot=(1 << 20) + 4)):
        assert _step(L, **bad) == A, bad
    assert lib.status_names(0x200) == ["BAD_WEIGHT"]


# ---- torch operators ---------------------------------------------------------------------------

def test_torch_operators_check_their_arguments_on_host_tensors():
    from asu_ascend_b200 import kv4

    bf, u8, i32 = torch.bfloat16, torch.uint8, torch.int32
    src, pool, slots = torch.zeros(4, 576, dtype=bf), torch.zeros(8, 416, dtype=u8), torch.zeros(4, dtype=i32)
    for args, text in (((src.float(), pool, slots), "bfloat16 or float16"),
                       ((src[:, :570], pool, slots), "576"),
                       ((torch.zeros(576, 4, dtype=bf).t(), pool, slots), "rows must be contiguous"),
                       ((src, pool[:, :400], slots), "416"),
                       ((src, pool.to(torch.int16), slots), "uint8"),
                       ((src, torch.zeros(8, 424, dtype=u8)[:, :416], slots), "multiples of 16"),
                       ((src, torch.zeros(1, 416, dtype=u8).expand(8, 416), slots), "must not overlap"),
                       ((src, pool[:0], slots), "no rows"),
                       ((src, pool, slots.long()), "int32"),
                       ((src, pool, slots[:3]), "one per row"),
                       ((src, pool[:3], None), "more rows than the pool"),
                       ((src.clone().requires_grad_(), pool, slots), "requires a gradient"),
                       ((src, pool, slots), "needs CUDA")):
        with pytest.raises(RuntimeError, match=text):
            kv4.pack_rows(*args)
    with pytest.raises(RuntimeError, match="needs CUDA"):
        kv4.unpack_rows(pool, slots)
    with pytest.raises(RuntimeError, match="contiguous"):
        kv4.unpack_rows(pool, torch.zeros(8, dtype=i32)[::2])
    q, sl = torch.zeros(2, 3, 576, dtype=bf), torch.zeros(2, 5, dtype=i32)
    for args, text in (((q.half(), pool, sl, 1.0), "bfloat16"), ((q[..., :512], pool, sl, 1.0), "576"),
                       ((q[0], pool, sl, 1.0), "576"),
                       ((torch.zeros(2, 129, 576, dtype=bf), pool, sl, 1.0), r"\[1, 128\]"),
                       ((q[:, :0], pool, sl, 1.0), r"\[1, 128\]"),
                       ((torch.zeros(2, 3, 1152, dtype=bf)[..., ::2], pool, sl, 1.0), "last dimension"),
                       ((q, pool.expand(3, 8, 416), sl, 1.0), "3 pools for 2 tokens"),
                       ((q, pool, sl[:1], 1.0), r"\[tokens, topk\]"), ((q, pool, sl.long(), 1.0), "int32"),
                       ((q, pool, torch.zeros(5, 2, dtype=i32).t(), 1.0), "rows must be contiguous"),
                       ((q, pool, torch.zeros(2, 16385, dtype=i32), 1.0), "16384"),
                       ((q, pool, sl, float("inf")), "scale"), ((q, pool, sl, 0.0), "scale"),
                       ((q, pool, sl, 1e-60), "scale"), ((q, pool, sl, 3e38), "scale"),
                       ((q.clone().requires_grad_(), pool, sl, 1.0), "requires a gradient"),
                       ((q, pool, sl, 1.0), "needs CUDA")):
        with pytest.raises((RuntimeError, ValueError), match=text):
            kv4.sparse_decode(*args)
    with torch.no_grad(), pytest.raises(RuntimeError, match="needs CUDA"):
        kv4.sparse_decode(q.clone().requires_grad_(), pool, sl, 1.0)


def test_torch_operators_on_meta_tensors():
    from asu_ascend_b200 import kv4

    m = torch.device("meta")
    q, pool = torch.empty(3, 7, 576, dtype=torch.bfloat16, device=m), torch.empty(9, 416, dtype=torch.uint8, device=m)
    got = kv4.sparse_decode(q, pool, torch.empty(3, 5, dtype=torch.int32, device=m), 0.1, weights=True)
    assert got.out.shape == (3, 7, 512) and got.lse.shape == (3, 7) and got.weights.shape == (3, 5)
    assert got.lse.dtype == torch.float32 and got.weights.dtype == torch.bfloat16
    assert kv4.unpack_rows(pool).shape == (9, 576)


def test_weight_slot_pools_check_their_arguments():
    from asu_ascend_b200.weight_pools import WeightSlotPools

    with pytest.raises(RuntimeError, match="CUDA"):
        WeightSlotPools(1, 100, 16, 4, 8, device="cpu")
    for bad in (dict(req_num=0), dict(slot_count=16385), dict(query_count=4097), dict(query_count=0),
                dict(free_target=-1), dict(decay=1.5), dict(decay=float("nan"))):
        kw = dict(req_num=1, key_space=100, slot_count=16, free_target=4, query_count=8, decay=1.0) | bad
        with pytest.raises((ValueError, RuntimeError)):
            z = torch.zeros
            R, S = kw["req_num"], kw["slot_count"]
            WeightSlotPools.from_state(z((R, 100), dtype=torch.int32), z((R, S), dtype=torch.int32), z((R, S)),
                                       z((R, S), dtype=torch.int32), z((R,), dtype=torch.int32),
                                       free_target=kw["free_target"], query_count=kw["query_count"], decay=kw["decay"])


def test_attention_workspace_is_bounded_whatever_the_call(lib):
    """256 MiB for the weights of the tokens that are done at once; the rest depends on the number of SMs alone."""
    size = lib.lib.asu_kv4_attention_workspace_bytes
    for heads in (1, 16, 17, 33, 64, 65, 128):
        for topk in (1, 130, 2048, 16384):
            for tokens in (1, 2, 500, 4096, 65535):
                bare, both = size(tokens, heads, topk, 0), size(tokens, heads, topk, 1)
                assert 0 <= bare <= 64 << 20 and bare <= both <= (256 + 64) << 20, (tokens, heads, topk, both)
    assert size(65535, 128, 0, 1) == size(65535, 128, 0, 0)


def test_tokens_that_no_ctas_share_need_no_workspace(lib):
    """One tile a token leaves nothing to join, whatever the number of SMs."""
    size = lib.lib.asu_kv4_attention_workspace_bytes
    for heads, tile in ((16, 128), (64, 128), (65, 64), (128, 64)):
        for tokens in (1, 7, 200, 5000):
            assert size(tokens, heads, tile, 0) == 0, (tokens, heads)


@pytest.mark.parametrize("device", [-7, 99])
def test_a_device_that_cannot_be_used_is_not_called_a_wrong_argument(lib, device):
    """The step's way to the device reports CUDA's error (no device, or an invalid one).  (A key space of 0, so that
    nothing can be launched.)"""
    from asu_ascend_b200 import ops

    rc = ops.weight_step(device, 0, None, *[16] * 5, None, None, 2, 0, 0.5, None, *[16] * 5, 4, 16, None, None, 1, 0, 8, 4, 4)
    assert rc > lib.ASU_ERR_CUDA_BASE
    with pytest.raises(lib.AsuError, match="device|driver|unknown|GPU"):
        lib.check(rc, "step")


def test_a_decode_without_its_attention_library_leaves_the_managed_cache_alone(monkeypatch):
    """Rows that need FlashMLA-sparse: where it is not installed the call fails before the resolver moves rows.  4-bit
    rows do not need it."""
    import sys

    from asu_ascend_b200 import sparse_mla

    calls = []
    monkeypatch.setitem(sys.modules, "vllm", None)
    monkeypatch.setattr(sparse_mla, "resolve_topk", lambda *a: calls.append(a) or torch.zeros(1, 4, dtype=torch.int32))
    q, topk = torch.zeros(1, 16, 576, dtype=torch.bfloat16), torch.zeros(1, 4, dtype=torch.int32)

    class Ctx:
        managed_kv_cache_0 = torch.zeros(64, 416, dtype=torch.uint8)

    with pytest.raises(ImportError):
        sparse_mla.sparse_mla_decode(q, Ctx, topk, topk[0], torch.zeros(2, 64, 576, dtype=torch.bfloat16), 0.1)
    assert not calls
    with pytest.raises(RuntimeError, match="needs CUDA"):
        sparse_mla.sparse_mla_decode(q, Ctx, topk, topk[0], torch.zeros(2, 64, 416, dtype=torch.uint8), 0.1)
    assert len(calls) == 1


def test_pools_of_one_row_or_one_token_may_have_any_stride_there():
    """A dimension of one element is never walked, so its stride does not count."""
    from asu_ascend_b200 import kv4

    bf, i32 = torch.bfloat16, torch.int32
    one = torch.zeros(416, 1, dtype=torch.uint8).t()
    assert one.shape == (1, 416) and one.stride() == (1, 1)
    odd = torch.zeros(3 * 425, dtype=torch.uint8).as_strided((1, 1, 416), (425, 424, 1))
    for call in (lambda: kv4.pack_rows(torch.zeros(1, 576, dtype=bf), one), lambda: kv4.unpack_rows(one),
                 lambda: kv4.sparse_decode(torch.zeros(1, 3, 576, dtype=bf), odd, torch.zeros(1, 5, dtype=i32), 1.0)):
        with pytest.raises(RuntimeError, match="needs CUDA"):
            call()
    for pool in (odd.expand(2, 1, 416), torch.zeros(2000, dtype=torch.uint8).as_strided((2, 1, 416), (424, 1, 1))):
        with pytest.raises(RuntimeError, match="needs CUDA" if pool.stride(0) == 0 else "multiples of 16"):
            kv4.sparse_decode(torch.zeros(2, 3, 576, dtype=bf), pool, torch.zeros(2, 5, dtype=i32), 1.0)


# ---- one wrong operand at a time ---------------------------------------------------------------

ALIGNED = dict(q=64, pool=64, slots=64, out=64, lse=64, ws=64, weights=64)


@pytest.mark.skipif(torch.cuda.is_available(), reason="a call without fault would launch on addresses that are none")
def test_the_aligned_calls_are_refused_for_want_of_a_device_alone(lib):
    assert _attention(lib.lib, **ALIGNED) > lib.ASU_ERR_CUDA_BASE
    assert lib.lib.asu_kv4_pack(None, 64, 0, 576, 4, None, 64, 8, 416, None) > lib.ASU_ERR_CUDA_BASE
    assert lib.lib.asu_kv4_unpack(None, 64, 8, 416, None, 4, 64, 576, None) > lib.ASU_ERR_CUDA_BASE


@pytest.mark.parametrize("bad", [
    dict(q=65), dict(pool=72), dict(pool=65), dict(pitch=424), dict(pitch=417), dict(pt=8), dict(pt=416 * 8 + 4),
    dict(slots=66), dict(out=48), dict(out=80), dict(lse=66), dict(ws=48), dict(weights=65)], ids=str)
def test_attention_rejects_each_operand_out_of_line(lib, bad):
    assert _attention(lib.lib, **(ALIGNED | bad)) == lib.ASU_ERR_ALIGN


@pytest.mark.parametrize("bad", [
    dict(tokens=-1), dict(tokens=65536), dict(heads=-1), dict(heads=129), dict(topk=-1), dict(topk=16385), dict(rows=-1),
    dict(rows=2**31), dict(qt=-1), dict(qh=-1), dict(st=-1), dict(pitch=400), dict(q=None), dict(out=None), dict(lse=None),
    dict(slots=None), dict(pool=None), dict(ws=None), dict(size=0), dict(scale=0.0), dict(scale=-1.0),
    dict(scale=float("inf")), dict(scale=float("nan")), dict(scale=3e38)], ids=str)
def test_attention_rejects_each_argument_out_of_range(lib, bad):
    assert _attention(lib.lib, **(ALIGNED | bad)) == lib.ASU_ERR_ARG


@pytest.mark.parametrize("bad,text", [
    (dict(R=0), "must be positive"), (dict(K=0), "must be positive"), (dict(S=0), "must be positive"),
    (dict(Q=0), "must be positive"), (dict(target=-1), "free_target >= 0"), (dict(S=16385), "slot_count <= 16384"),
    (dict(Q=4097), "query_count <= 4096"), (dict(decay=1.5), "decay"), (dict(decay=-0.1), "decay"),
    (dict(decay=float("nan")), "decay"), (dict(), None)], ids=str)
def test_weight_slot_pools_reject_each_argument(bad, text):
    """ValueErrors of the sizes, which come before the device's RuntimeError (the last case: nothing else is wrong)."""
    from asu_ascend_b200.weight_pools import WeightSlotPools

    a = dict(R=1, K=100, S=16, Q=8, target=4, decay=1.0) | bad
    i32 = dict(dtype=torch.int32)
    state = (torch.zeros(a["R"], a["K"], **i32), torch.zeros(a["R"], a["S"], **i32), torch.zeros(a["R"], a["S"]),
             torch.zeros(a["R"], a["S"], **i32), torch.zeros(a["R"], **i32))
    with pytest.raises(RuntimeError if text is None else ValueError, match=text or "lives in HBM"):
        WeightSlotPools.from_state(*state, free_target=a["target"], query_count=a["Q"], decay=a["decay"])


@pytest.mark.parametrize("which", range(5))
def test_weight_slot_pools_reject_each_state_tensor(which):
    from asu_ascend_b200.weight_pools import WeightSlotPools

    names = ("token_to_slot", "slot_to_token", "score", "free_stack", "free_count")
    shapes = ((2, 100), (2, 16), (2, 16), (2, 16), (2,))
    state = [torch.zeros(s, dtype=torch.float32 if n == "score" else torch.int32) for n, s in zip(names, shapes)]
    good = state[which]
    for wrong in (good.to(torch.float64), torch.stack([good, good], -1)[..., 0], good.to("meta")):
        state[which] = wrong
        with pytest.raises(RuntimeError, match="on meta" if which == 0 and wrong.is_meta else f"{names[which]} must be"):
            WeightSlotPools.from_state(*state, free_target=4, query_count=8)
