"""Slot pools that evict by accumulated attention weight, bit for bit against the serial oracle: slots,
masks, evicted keys, scores and the whole state over several steps; odd inputs; and the pools together
with the 4-bit cache and the swap-in."""

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def WeightSlotPools():
    import asu_ascend_b200

    asu_ascend_b200.load()
    from asu_ascend_b200.weight_pools import WeightSlotPools

    return WeightSlotPools


def compare(pools, oracle, out, results):
    slot, hit, inst = out.slot.cpu().numpy(), out.hit.cpu().numpy(), out.install.cpu().numpy()
    ev, evn = out.evicted.cpu().numpy(), out.evicted_count.cpu().numpy()
    score, s2t = pools.score.cpu().numpy(), pools.slot_to_token.cpu().numpy()
    stack, free = pools.free_stack.cpu().numpy(), pools.free_count.cpu().numpy()
    for r, (p, (o_slot, o_hit, o_inst, o_ev)) in enumerate(zip(oracle, results)):
        assert slot[r].tolist() == o_slot, r
        assert hit[r].tolist() == o_hit and inst[r].tolist() == o_inst, r
        assert evn[r] == len(o_ev) and ev[r, :evn[r]].tolist() == o_ev, r
        assert (ev[r, evn[r]: p.target] == -1).all()
        assert np.array_equal(score[r].view(np.uint32), p.score.view(np.uint32)), r
        assert s2t[r].tolist() == p.slot_key and stack[r, :free[r]].tolist() == p.stack, r
        row = np.full(pools.key_space, -1, np.int32)
        for k, s in p.key_slot.items():
            row[k] = s
        assert np.array_equal(pools.token_to_slot[r].cpu().numpy(), row), r


def drive(pools, R, K, S, Q, target, decay, steps, seed, dtype=torch.float32, repeats=False, bad=False, keep=None, n_last=None):
    rng = np.random.default_rng(seed)
    oracle = [O.WeightPool(S, target, decay) for _ in range(R)]
    last_s = last_w = None
    hot = rng.permutation(K)[: max(1, min(K, S // 2))]
    for step in range(steps):
        q = np.empty((R, Q), np.int32)
        for r in range(R):
            pick = np.concatenate([rng.choice(hot, Q), rng.integers(0, K, Q)])
            q[r] = rng.choice(pick, Q, replace=repeats) if repeats else (
                rng.permutation(np.unique(np.concatenate([pick, rng.permutation(K)[:Q]])))[:Q])
        if bad:
            q[0, 0], q[-1, -1] = -1, K + 5
        kf = None if keep is None else rng.integers(0, K, R).astype(np.int32)
        args = [torch.from_numpy(q).to(DEV)]
        if last_s is not None:
            args += [torch.from_numpy(last_s).to(DEV), last_w.to(DEV)]
        out = pools.step(*args, keep_from=None if kf is None else torch.from_numpy(kf).to(DEV))
        results = [p.step(q[r].tolist(), () if last_s is None else last_s[r].tolist(),
                          () if last_s is None else last_w[r].float().tolist(),
                          2**31 - 1 if kf is None else int(kf[r]), K) for r, p in enumerate(oracle)]
        compare(pools, oracle, out, results)
        last_s = out.slot.cpu().numpy()
        if n_last is not None:
            last_s = np.ascontiguousarray(last_s[:, rng.integers(0, Q, n_last)])
        # few distinct weights: ties at every threshold
        last_w = torch.from_numpy((rng.integers(0, 6, last_s.shape) / 4).astype(np.float32)).to(dtype)
    return oracle


@pytest.mark.parametrize("R,K,S,Q,target,decay,dtype,repeats,keep,n_last", [
    (1, 50, 8, 3, 4, 0.5, torch.float32, False, None, None),
    (3, 300, 64, 16, 20, 0.9, torch.bfloat16, False, None, None),
    (2, 5000, 1001, 333, 301, 0.98, torch.float32, False, True, None),
    (4, 400, 37, 20, 30, 1.0, torch.float32, True, None, None),     # repeats in the top-k, shortages
    (2, 3000, 257, 100, 120, 0.0, torch.bfloat16, True, True, 40),  # no memory; fewer weights than keys
    (1, 1, 1, 1, 1, 1.0, torch.float32, False, None, None),
    (2, 9000, 2049, 700, 700, 0.97, torch.float32, False, None, None),
    (1, 40000, 8200, 2048, 2048, 0.97, torch.bfloat16, False, None, None),
    (1, 60000, 16384, 4096, 4096, 0.97, torch.float32, True, None, 4096),
])
def test_steps_match_the_oracle(WeightSlotPools, R, K, S, Q, target, decay, dtype, repeats, keep, n_last):
    pools = WeightSlotPools(R, K, S, target, Q, decay=decay, device=DEV)
    oracle = drive(pools, R, K, S, Q, target, decay, 6, R + S + Q, dtype, repeats, False, keep, n_last)
    pools.check_status()
    t = pools.totals()
    assert t["hits"] + t["misses"] == 6 * R * Q and t["installs"] - t["evictions"] == sum(len(p.key_slot) for p in oracle)


def test_bad_keys_are_skipped_and_reported(WeightSlotPools):
    pools = WeightSlotPools(2, 300, 64, 20, 16, decay=0.9, device=DEV)
    drive(pools, 2, 300, 64, 16, 20, 0.9, 4, 5, bad=True)
    with pytest.raises(RuntimeError, match="BAD_QUERY"):
        pools.check_status()


def test_bad_weights_and_stale_slots(WeightSlotPools):
    pools = WeightSlotPools(1, 100, 8, 2, 4, decay=1.0, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    pools.step(torch.tensor([[1, 2, 3, 4]], **i32))
    last = torch.tensor([[0, 1, 2, 3, 0, 7, -1]], **i32)
    w = torch.tensor([[1.0, -1.0, float("nan"), float("inf"), 0.25, 5.0, 9.0]], device=DEV)
    out = pools.step(torch.tensor([[1, 2, 3, 4]], **i32), last, w)
    assert out.hit.all() and pools.score[0].tolist() == [1.25, 0, 0, 0, 0, 0, 0, 0]  # slot 7 holds no token
    with pytest.raises(RuntimeError, match="BAD_WEIGHT"):
        pools.check_status()
    pools.status.zero_()
    pools.step(torch.tensor([[1, 2, 3, 4]], **i32), torch.tensor([[8, -5]], **i32), torch.ones(1, 2, device=DEV))
    with pytest.raises(RuntimeError, match="BAD_QUERY"):
        pools.check_status()
    pools.status.zero_()
    pools.free_count.fill_(9)  # corrupt: more free slots than slots
    before = [t.clone() for t in (pools.token_to_slot, pools.slot_to_token, pools.score, pools.free_stack)]
    out = pools.step(torch.tensor([[1, 2, 3, 4]], **i32))
    assert (out.slot == -1).all() and not out.install.any() and not out.hit.any() and int(out.evicted_count) == 0
    for a, b in zip(before, (pools.token_to_slot, pools.slot_to_token, pools.score, pools.free_stack)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="BAD_STATE"):
        pools.check_status()


def test_nothing_may_leave(WeightSlotPools):
    """Every resident token is asked for or kept: no eviction, then shortages."""
    pools = WeightSlotPools(1, 100, 4, 4, 4, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    pools.step(torch.tensor([[10, 11, 12, 13]], **i32))
    out = pools.step(torch.tensor([[10, 11, 12, 13]], **i32))
    assert out.hit.all() and int(out.evicted_count) == 0
    out = pools.step(torch.tensor([[50, 51, 10, 11]], **i32), keep_from=torch.tensor([12], **i32))
    assert out.slot.tolist() == [[-1, -1, 0, 1]] and int(out.evicted_count) == 0
    assert pools.totals()["shortages"] == 2


def test_step_refuses_wrong_tensors(WeightSlotPools):
    pools = WeightSlotPools(2, 100, 16, 4, 8, device=DEV)
    q, w = torch.zeros(2, 8, dtype=torch.int32, device=DEV), torch.zeros(2, 8, device=DEV)
    for args, kw, text in (((q.cpu(),), {}, "query"), ((q[:1],), {}, "query must be"), ((q, q), {}, "go together"),
                           ((q, q, w.half()), {}, "last_weight"), ((q, q, w[:, :4].contiguous()), {}, "both be"),
                           ((q, q.long(), w), {}, "last_slot"), ((q, q[:, ::2], w[:, ::2]), {}, "last_slot"),
                           ((q,), dict(keep_from=q[0]), "keep_from"),
                           ((q, q.repeat(1, 513), w.repeat(1, 513)), {}, "4096")):
        with pytest.raises(RuntimeError, match=text):
            pools.step(*args, **kw)


def test_step_refuses_output_buffers_of_other_pools(WeightSlotPools):
    pools = WeightSlotPools(2, 100, 16, 4, 8, device=DEV)
    q = torch.zeros(2, 8, dtype=torch.int32, device=DEV)
    pools.step(q, out=pools.new_output())
    for other in (WeightSlotPools(2, 100, 16, 4, 7, device=DEV), WeightSlotPools(1, 100, 16, 4, 8, device=DEV),
                  WeightSlotPools(2, 100, 16, 3, 8, device=DEV)):
        with pytest.raises(RuntimeError, match="new_output"):
            pools.step(q, out=other.new_output())
    out = pools.new_output()
    out.hit = out.hit.to(torch.int32)
    with pytest.raises(RuntimeError, match="out.hit"):
        pools.step(q, out=out)


@pytest.mark.parametrize("n,names", [(4096, 1), (4096, 3), (1500, 700), (33, 2)])
def test_many_weights_of_one_slot_add_up_in_their_order(WeightSlotPools, n, names):
    """Every rounding counts: weights of many sizes, and the sum in the entries' order bit for bit."""
    S = 1024
    pools = WeightSlotPools(1, 5000, S, 0, 1024, decay=0.75, device=DEV)
    keys = torch.arange(S, dtype=torch.int32, device=DEV).view(1, S)
    pools.step(keys)
    rng = np.random.default_rng(n + names)
    pools.score.copy_(torch.from_numpy(rng.random((1, S)).astype(np.float32)))
    score = (pools.score[0].cpu().numpy() * np.float32(0.75)).astype(np.float32)
    last = rng.permutation(S)[:names][rng.integers(0, names, n)].astype(np.int32)
    w = np.exp2(rng.uniform(-20, 3, n)).astype(np.float32)
    for s, x in zip(last, w):
        score[s] = np.float32(score[s] + x)
    pools.step(keys, torch.from_numpy(last).view(1, n).to(DEV), torch.from_numpy(w).view(1, n).to(DEV))
    assert np.array_equal(pools.score[0].cpu().numpy().view(np.uint32), score.view(np.uint32))
    pools.check_status()


def test_scores_that_cannot_be_count_as_zero_and_are_reported(WeightSlotPools):
    """Negative and NaN scores of a state that someone else wrote: the lowest, by slot, and the status says so;
    infinite ones are the last to leave."""
    pools = WeightSlotPools(1, 100, 8, 3, 8, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    pools.step(torch.arange(8, **i32).view(1, 8))
    pools.score.copy_(torch.tensor([[float("inf"), 1.0, -3.0, 2.0, float("nan"), -0.0, 0.5, float("inf")]], device=DEV))
    out = pools.step(torch.full((1, 8), 50, **i32))
    assert out.evicted[0].tolist() == [2, 4, 5] and int(out.evicted_count) == 3
    assert pools.score[0].tolist() == [float("inf"), 1, 0, 2, 0, 0, 0.5, float("inf")]
    with pytest.raises(RuntimeError, match="BAD_STATE"):
        pools.check_status()
    pools.status.zero_()
    pools.score.copy_(torch.full((1, 8), float("inf"), device=DEV))
    out = pools.step(torch.full((1, 8), 60, **i32))
    assert int(out.evicted_count) == 1 and out.evicted[0, 0] == 0  # free 2 of 3: one more, the lowest slot


def test_graph_replay_and_the_step_writing_over_its_last_slots(WeightSlotPools):
    """One captured step whose last_slot is its own output buffer, against eager steps with copies."""
    R, K, S, Q, target = 3, 2000, 256, 64, 80
    a, b = (WeightSlotPools(R, K, S, target, Q, decay=0.9, device=DEV) for _ in range(2))
    rng = np.random.default_rng(2)
    query = torch.zeros(R, Q, dtype=torch.int32, device=DEV)
    weight = torch.zeros(R, Q, dtype=torch.bfloat16, device=DEV)
    oa = a.new_output()
    oa.slot.fill_(-1)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            a.step(query, oa.slot, weight, out=oa)
    torch.cuda.synchronize()
    last = torch.full((R, Q), -1, dtype=torch.int32, device=DEV)
    for step in range(8):
        query.copy_(torch.from_numpy(np.stack([rng.permutation(400 + 100 * step)[:Q] for _ in range(R)]).astype(np.int32)))
        weight.copy_(torch.from_numpy(rng.random((R, Q)).astype(np.float32)))
        torch.cuda.synchronize()
        g.replay()
        ob = b.step(query, last, weight)
        torch.cuda.synchronize()
        for x, y in ((oa.slot, ob.slot), (oa.hit, ob.hit), (oa.install, ob.install), (oa.evicted, ob.evicted),
                     (a.score, b.score), (a.slot_to_token, b.slot_to_token), (a.free_count, b.free_count)):
            assert torch.equal(x, y)
        last = ob.slot.clone()
    assert int(a.stats[:, 4].sum()) > 0


def test_the_cache_the_attention_and_the_eviction_together(WeightSlotPools):
    """A decode loop over a host pool of 4-bit rows: step, swap-in, attention with weights, and the next step
    with those weights; every output against the oracle, over enough steps for evictions."""
    from asu_ascend_b200 import kv4
    from asu_ascend_b200.host_pool import HostRowPool, check_status

    R, K, S, Q, target, H = 3, 600, 160, 48, 64, 24
    g = torch.Generator().manual_seed(4)
    x = torch.randn(R * K, 576, generator=g).to(torch.bfloat16)
    packed = kv4.new_pool(R * K, device=DEV)
    kv4.pack_rows(x.to(DEV), packed)
    host = HostRowPool(R * K, kv4.ROW_BYTES)
    host.writeback_range(packed, 0)
    rec = torch.arange(R * K, dtype=torch.int32, device=DEV).view(R, K)
    pools = WeightSlotPools(R, K, S, target, Q, decay=0.9, device=DEV)
    oracle = [O.WeightPool(S, target, 0.9) for _ in range(R)]
    managed = kv4.new_pool(R, S, device=DEV)
    status = torch.zeros(R, dtype=torch.int32, device=DEV)
    rows = packed.cpu().numpy().reshape(R, K, 416)
    rng = np.random.default_rng(6)
    last = weights = None
    for step in range(7):
        q_ids = np.stack([rng.permutation(200 + 60 * step)[:Q] for _ in range(R)]).astype(np.int32)
        topk = torch.from_numpy(q_ids).to(DEV)
        out = pools.step(topk, last, weights)
        results = [p.step(q_ids[r].tolist(), () if last is None else last[r].tolist(),
                          () if last is None else weights[r].float().tolist()) for r, p in enumerate(oracle)]
        compare(pools, oracle, out, results)
        host.swapin(rec, topk, out.slot, out.install, managed, status=status)
        q = torch.randn(R, H, 576, generator=g).to(torch.bfloat16)
        got = kv4.sparse_decode(q.to(DEV), managed, out.slot, 0.07, weights=True)
        for r in range(R):
            o, l, w, mag, smag = O.attention(q[r].float().numpy(), rows[r], q_ids[r], 0.07)
            ds = (576 * 2.0**-23 + 2.0**-22) * smag
            lim = (2.0**-8 + 2 * ds[:, None] + 2 * 2.0**-16) * mag
            assert (np.abs(got.out[r].float().cpu().numpy() - o) <= lim + 2.0**-8 * (np.abs(o) + lim)).all()
            assert (np.abs(got.weights[r].float().cpu().numpy() - w) <= w * (2 * 2.0**-8 + 2 * ds.max() + 2.0**-16)
                    * (1 + 2.0**-7) + 2.0**-32 * H).all()
        last, weights = out.slot.clone(), got.weights
    check_status(status, "swapin")
    pools.check_status()
    assert pools.totals()["evictions"] > 0
    host.close()


def test_a_refused_row_lists_no_evicted_keys(WeightSlotPools):
    """free_count out of range after a step that evicted: that row's outputs say that nothing left, the whole list."""
    pools = WeightSlotPools(2, 100, 8, 3, 4, device=DEV)
    i32 = dict(dtype=torch.int32, device=DEV)
    keys = torch.tensor([[0, 1, 2, 3], [5, 6, 7, 8]], **i32)
    for step in range(3):
        out = pools.step(keys + 10 * step)
    assert out.evicted_count.tolist() == [3, 3] and (out.evicted >= 0).all()
    pools.free_count[1] = -1
    out = pools.step(keys + 30)
    assert out.evicted_count.tolist() == [3, 0]
    assert (out.evicted[0] >= 0).all() and (out.evicted[1] == -1).all()
    with pytest.raises(RuntimeError, match="BAD_STATE"):
        pools.check_status()
