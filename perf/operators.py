"""The 4-bit MLA cache and the attention-weight slot pools: what their calls are timed on.

Three operators, used together in a sparse-attention decode step over a managed cache:

``rows``    latent rows written into a 4-bit pool and read back (the cache's write and read side)
``decode``  sparse MLA attention of decode tokens over the 4-bit rows that their slots name
``step``    one step of slot pools that evict by accumulated attention weight

A 4-bit row is 416 bytes: 512 latent values in 4 bits (256 bytes), their 32 group scales (one byte
for 16 values), and 64 position-encoded values in bf16 (128 bytes).  Value i of a group is
(n - 8) * s with n in 1..15.  A scale byte b is the number (1 + (b & 7) / 8) * 2**((b >> 3) - 18).
Eight values share a 32-bit word: value 2j is nibble j, value 2j + 1 is nibble j + 4.
"""

import math

import torch

own = False

LATENT, ROPE, GROUP = 512, 64, 16
DIM = LATENT + ROPE
ROW = LATENT // 2 + LATENT // GROUP + 2 * ROPE
BIAS = 18
CODES, SCALES = slice(0, 256), slice(256, 288)
SCALE = 192.0 ** -0.5  # of a 128 + 64 wide attention head before its latent form
DECAY = 0.98
BATCHES = 8


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # one token's row appended to the cache, and read back
        {"name": "rows-1", "op": "rows", "n": 1, "dtype": "bf16", "pad": 0, "pool": 8192},
        # a chunk of a prompt from an fp16 buffer with wider rows, into scattered slots
        {"name": "rows-4099-fp16-strided", "op": "rows", "n": 4099, "dtype": "fp16", "pad": 64, "pool": 10240},
        # half of a 128K-token prompt
        {"name": "rows-65536", "op": "rows", "n": 65536, "dtype": "bf16", "pad": 0, "pool": 131072},
        # one request at the start of its answer, the heads of one rank of eight
        {"name": "decode-1x16x100", "op": "decode", "tokens": 1, "heads": 16, "topk": 100, "slots": 2048,
         "own_pools": False, "weights": False, "ragged": False},
        # the single-request decode path: all heads, the managed cache of 8192 + 2048 slots
        {"name": "decode-1x128x2048", "op": "decode", "tokens": 1, "heads": 128, "topk": 2048, "slots": 10240,
         "own_pools": False, "weights": True, "ragged": False},
        # a batch of 128 requests, each with its own pool of 8192 slots, the heads of one rank of eight
        {"name": "decode-128x16x2048", "op": "decode", "tokens": 128, "heads": 16, "topk": 2048, "slots": 8192,
         "own_pools": True, "weights": False, "ragged": False},
        # the same with all heads, and the weights that the eviction accumulates
        {"name": "decode-128x128x2048", "op": "decode", "tokens": 128, "heads": 128, "topk": 2048, "slots": 8192,
         "own_pools": True, "weights": True, "ragged": False},
        # requests of different lengths (padded with -1, one without any key) and an odd head count
        {"name": "decode-37x24x777-ragged", "op": "decode", "tokens": 37, "heads": 24, "topk": 777, "slots": 5003,
         "own_pools": True, "weights": True, "ragged": True},
        # several tokens over one shared pool, half of the heads
        {"name": "decode-61x64x1024-shared", "op": "decode", "tokens": 61, "heads": 64, "topk": 1024, "slots": 10240,
         "own_pools": False, "weights": False, "ragged": False},
        # one request's layer: 8192 resident slots and 2048 free ones
        {"name": "step-1x10240", "op": "step", "requests": 1, "keys": 131072, "slots": 10240, "topk": 2048,
         "target": 2048, "keep": 0},
        # odd sizes, with the latest positions kept
        {"name": "step-37x1001-keep", "op": "step", "requests": 37, "keys": 70001, "slots": 1001, "topk": 333,
         "target": 301, "keep": 4096},
        # the resolver's default batch
        {"name": "step-128x8192", "op": "step", "requests": 128, "keys": 131072, "slots": 8192, "topk": 2048,
         "target": 2048, "keep": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rows", "decode", "decode", "step"])
    if op == "rows":
        n = _log(rng, 1, 65536)
        return {"op": op, "n": n, "dtype": rng.choice(["bf16", "fp16"]), "pad": rng.choice([0, 0, 8, 64, 72]),
                "pool": n + _log(rng, 1, 65536)}
    if op == "decode":
        topk = _log(rng, 1, 2048)
        return {"op": op, "tokens": _log(rng, 1, 128), "heads": _log(rng, 1, 128), "topk": topk,
                "slots": topk + _log(rng, 1, 6144), "own_pools": rng.random() < 0.5,
                "weights": rng.random() < 0.5, "ragged": rng.random() < 0.5}
    slots = _log(rng, 64, 10240)
    topk = max(1, min(2048, int(slots * rng.uniform(0.05, 0.3))))
    return {"op": op, "requests": _log(rng, 1, 128), "keys": _log(rng, 4 * slots, 131072), "slots": slots,
            "topk": topk, "target": max(topk, int(slots * rng.uniform(0.15, 0.3))),
            "keep": rng.choice([0, 0, _log(rng, 16, 4096)])}


# ---- inputs ------------------------------------------------------------------------------------

def _gen(seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed) * 1000003 + 12345)
    return g, dev


def _latents(n, g, dev):
    """Rows as a cache holds them: normed latents whose channels differ in size, and rope parts."""
    channel = torch.exp(0.6 * torch.randn(DIM, generator=g, device=dev))
    channel[LATENT:] = 1.5
    return torch.randn(n, DIM, generator=g, device=dev) * channel


def _pack(x):
    """Rows [n, 576] of 32-bit floats (holding 16-bit values) -> bytes [n, 416]."""
    n = x.shape[0]
    lat = x[:, :LATENT].reshape(n, LATENT // GROUP, GROUP)
    top = lat.abs().amax(-1)
    bits = (top / torch.full_like(top, 7.0)).view(torch.int32)  # by a tensor: a number would be multiplied by its reciprocal
    bits = bits + 0x7FFFF + ((bits >> 20) & 1)  # to three bits behind the point, ties to even
    byte = ((bits >> 20) - ((127 - BIAS) << 3)).clamp(0, 255)
    s = ((byte << 20) + ((127 - BIAS) << 23)).view(torch.float32)
    nib = (torch.round(lat / s[..., None]).clamp(-7, 7) + 8).to(torch.int32).reshape(n, LATENT // 8, 4, 2)
    low = nib[:, :, ::2] | (nib[:, :, 1::2] << 4)  # [n, 64, 2, 2]: byte of the pair of pairs, even / odd values
    codes = low.permute(0, 1, 3, 2).reshape(n, LATENT // 2).to(torch.uint8)
    rope = x[:, LATENT:].to(torch.bfloat16).contiguous().view(torch.uint8)
    return torch.cat([codes, byte.to(torch.uint8), rope], 1)


def _unpack(b):
    """Bytes [..., 416] -> values [..., 576] in 32 bits."""
    lead = b.shape[:-1]
    c = b[..., CODES].reshape(*lead, LATENT // 8, 2, 2)
    nib = torch.stack([c & 15, c >> 4], -1)  # [..., word, even / odd, byte, nibble of the byte]
    val = nib.reshape(*lead, LATENT // 8, 2, 4).transpose(-1, -2).reshape(*lead, LATENT // GROUP, GROUP)
    byte = b[..., SCALES].to(torch.int32)
    s = ((byte << 20) + ((127 - BIAS) << 23)).view(torch.float32)
    lat = ((val.to(torch.float32) - 8.0) * s[..., None]).reshape(*lead, LATENT)
    rope = b[..., 288:].contiguous().view(torch.bfloat16).to(torch.float32)
    return torch.cat([lat, rope], -1)


def _distinct(rows, of, n, g, dev):
    """[rows, n] distinct numbers below `of` in each row, in no order."""
    return torch.rand(rows, of, generator=g, device=dev).argsort(1)[:, :n]


def prepare(case, seed):
    g, dev = _gen(seed)
    if case["op"] == "rows":
        n, dt = case["n"], {"bf16": torch.bfloat16, "fp16": torch.float16}[case["dtype"]]
        buf = torch.zeros(n, DIM + case["pad"], device=dev, dtype=dt)
        src = buf[:, :DIM]
        src.copy_(_latents(n, g, dev))
        pool = torch.randint(0, 256, (case["pool"], ROW), generator=g, device=dev, dtype=torch.uint8)
        slots = torch.randperm(case["pool"], generator=g, device=dev)[:n].to(torch.int32)
        return {"op": "rows", "src": src, "pool": pool, "slots": slots}
    if case["op"] == "decode":
        T, H, K, S = case["tokens"], case["heads"], case["topk"], case["slots"]
        pools = T if case["own_pools"] else 1
        pool = torch.empty(pools, S, ROW, device=dev, dtype=torch.uint8)
        for i in range(pools):
            pool[i] = _pack(_latents(S, g, dev).to(torch.bfloat16).float())
        slots = _distinct(T, S, K, g, dev).to(torch.int32)
        if case["ragged"]:  # the last keys of a row are padding; a few holes; one row has no key at all
            length = torch.randint(0, K + 1, (T, 1), generator=g, device=dev)
            hole = torch.rand(T, K, generator=g, device=dev) < 0.03
            slots[(torch.arange(K, device=dev) >= length) | hole] = -1
            slots[T // 2] = -1
        q = (torch.randn(T, H, DIM, generator=g, device=dev)).to(torch.bfloat16)
        return {"op": "decode", "q": q, "pool": pool if case["own_pools"] else pool[0], "slots": slots,
                "weights": case["weights"]}
    R, K, S, Q, target = case["requests"], case["keys"], case["slots"], case["topk"], case["target"]
    # keys that each step asks for: three quarters from a hot set that fits, the rest seen once a cycle
    hot = min(S // 2, K // 2)
    n_hot = min(hot, Q - Q // 4)
    n_cold = Q - n_hot
    perm = _distinct(R, K, min(K, hot + n_cold * BATCHES), g, dev).to(torch.int32)
    query = []
    for b in range(BATCHES):
        h = perm.gather(1, _distinct(R, hot, n_hot, g, dev))
        at = hot + (b * n_cold + torch.arange(n_cold, device=dev)) % max(1, perm.shape[1] - hot)
        both = torch.cat([h, perm[:, at]], 1) if n_cold else h
        mix = torch.rand(R, Q, generator=g, device=dev).argsort(1)
        query.append(both.gather(1, mix).contiguous())
    # weights of a step, as attention gives them: a few large ones, summed over 16 heads
    weight = torch.softmax(3.0 * torch.randn(BATCHES, R, Q, generator=g, device=dev), -1).mul(16.0).to(torch.bfloat16)
    live = min(S, S - target + n_cold, perm.shape[1])  # residents before the first step
    flat = torch.full((R * K + 1,), -1, device=dev, dtype=torch.int32)  # one entry more, for the plain form's use
    t2s = flat[: R * K].view(R, K)
    slot_ids = torch.arange(live, device=dev, dtype=torch.int32).expand(R, live)
    s2t = torch.full((R, S), -1, device=dev, dtype=torch.int32)
    s2t[:, :live] = perm[:, :live]
    t2s.scatter_(1, perm[:, :live].long(), slot_ids)
    score = torch.zeros(R, S, device=dev)
    score[:, :live] = torch.empty(R, live, device=dev).exponential_(generator=g)
    stack = torch.full((R, S), -1, device=dev, dtype=torch.int32)
    if live < S:
        stack[:, : S - live] = torch.arange(S - 1, live - 1, -1, device=dev, dtype=torch.int32)
    keep = None
    if case["keep"]:
        keep = torch.full((R,), max(0, K - case["keep"]), device=dev, dtype=torch.int32)
    return {"op": "step", "flat": flat, "token_to_slot": t2s, "slot_to_token": s2t, "score": score,
            "free_stack": stack, "free_count": torch.full((R,), S - live, device=dev, dtype=torch.int32),
            "keep_from": keep, "query": query, "weight": list(weight.unbind(0)), "target": target, "at": 0,
            "last_slot": torch.full((R, Q), -1, device=dev, dtype=torch.int32)}


# ---- plain forms -------------------------------------------------------------------------------

def _rows_plain(st):
    at = st["slots"].long()
    st["pool"][at] = _pack(st["src"].float())
    return {"rows": _unpack(st["pool"][at]).to(torch.bfloat16)}


def _decode_plain(st):
    q, pool, slots = st["q"].float(), st["pool"], st["slots"].long()
    valid = slots >= 0
    at = slots.clamp(min=0)
    if pool.dim() == 3:
        rows = pool[torch.arange(pool.shape[0], device=pool.device)[:, None], at]
    else:
        rows = pool[at]
    kv = _unpack(rows)
    s = torch.matmul(q, kv.transpose(1, 2)) * SCALE
    s = s.masked_fill(~valid[:, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m.masked_fill(m == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    got = {"out": torch.matmul(p, kv[..., :LATENT]).to(torch.bfloat16), "lse": (m + torch.log(total))[..., 0]}
    if st["weights"]:
        got["weights"] = p.sum(1).to(torch.bfloat16)
    return got


def _step_plain(st, query, weight):
    t2s, s2t, score, stack, free = (st[k] for k in ("token_to_slot", "slot_to_token", "score", "free_stack", "free_count"))
    R, K = t2s.shape
    S, Q, target = s2t.shape[1], query.shape[1], min(st["target"], s2t.shape[1])
    dev = t2s.device
    base = torch.arange(R, device=dev)[:, None] * K
    none = R * K
    # the last step's weights
    last = st["last_slot"].long()
    score.mul_(DECAY)
    score.scatter_add_(1, last.clamp(min=0), weight.float().masked_fill(last < 0, 0.0))
    # who may go
    ok = (query >= 0) & (query < K)
    q = query.clamp(0, K - 1).long()
    found = t2s.gather(1, q)
    hit = ok & (found >= 0)
    asked = torch.zeros(R, S + 1, device=dev, dtype=torch.bool)
    asked.scatter_(1, torch.where(hit, found.long(), S), True)
    may = (s2t >= 0) & ~asked[:, :S]
    if st["keep_from"] is not None:
        may &= s2t < st["keep_from"][:, None]
    n = torch.minimum((target - free).clamp(min=0), may.sum(1))
    order = score.masked_fill(~may, math.inf).sort(dim=1, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, torch.arange(S, device=dev).expand(R, S))
    gone = may & (rank < n[:, None])
    # their slots in rising order onto the stack
    to = gone.cumsum(1) - 1
    wide = torch.cat([stack, stack[:, :1]], 1)
    ids = torch.arange(S, device=dev, dtype=torch.int32).expand(R, S)
    wide.scatter_(1, torch.where(gone, free[:, None] + to, S), ids)
    stack.copy_(wide[:, :S])
    evicted = torch.full((R, target + 1), -1, device=dev, dtype=torch.int32)
    evicted.scatter_(1, torch.where(gone, to, target), s2t)
    st["flat"][torch.where(gone, base + s2t, none)] = -1
    s2t.masked_fill_(gone, -1)
    score.masked_fill_(gone, 0.0)
    free1 = free + n
    # misses: the first position of each key takes a slot, in query order
    miss = ok & ~hit
    by = torch.where(miss, q, K).sort(dim=1, stable=True)
    new = torch.ones(R, Q, device=dev, dtype=torch.bool)
    new[:, 1:] = by.values[:, 1:] != by.values[:, :-1]
    first = torch.empty_like(new).scatter_(1, by.indices, new) & miss
    turn = first.cumsum(1) - 1
    inst = first & (turn < free1[:, None])
    slot = stack.gather(1, (free1[:, None] - 1 - turn).clamp(0, S - 1))
    st["flat"][torch.where(inst, base + q, none)] = torch.where(inst, slot, -1)
    wide = torch.cat([s2t, s2t[:, :1]], 1)
    wide.scatter_(1, torch.where(inst, slot.long(), S), query)
    s2t.copy_(wide[:, :S])
    out = t2s.gather(1, q).masked_fill(~ok, -1)
    free.copy_(free1 - torch.minimum(first.sum(1), free1))
    return {"slot": out, "hit": hit | (miss & ~first & (out >= 0)), "install": inst, "evicted": evicted[:, :target],
            "evicted_count": n.to(torch.int32)}


def run(state):
    if state["op"] == "rows":
        if own:
            from asu_ascend_b200 import kv4

            kv4.pack_rows(state["src"], state["pool"], state["slots"])
            return {"rows": kv4.unpack_rows(state["pool"], state["slots"])}
        return _rows_plain(state)
    if state["op"] == "decode":
        if own:
            from asu_ascend_b200 import kv4

            got = kv4.sparse_decode(state["q"], state["pool"], state["slots"], SCALE, weights=state["weights"])
            return {"out": got.out, "lse": got.lse} | ({"weights": got.weights} if state["weights"] else {})
        return _decode_plain(state)
    at = state["at"]
    state["at"] = (at + 1) % BATCHES
    query, weight = state["query"][at], state["weight"][at]
    if own:
        if "pools" not in state:
            from asu_ascend_b200.weight_pools import WeightSlotPools

            state["pools"] = WeightSlotPools.from_state(
                state["token_to_slot"], state["slot_to_token"], state["score"], state["free_stack"],
                state["free_count"], free_target=state["target"], query_count=query.shape[1], decay=DECAY)
        o = state["pools"].step(query, state["last_slot"], weight, keep_from=state["keep_from"])
        got = {"slot": o.slot, "hit": o.hit, "install": o.install, "evicted": o.evicted, "evicted_count": o.evicted_count}
    else:
        got = _step_plain(state, query, weight)
    state["last_slot"] = got["slot"]
    return got | {k: state[k] for k in ("token_to_slot", "slot_to_token", "score", "free_stack", "free_count")}


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    if case["op"] == "rows":
        n = case["n"]
        return {"bytes": n * (2 * DIM + ROW + ROW + 2 * DIM + 2 * 4), "flops": 0}
    if case["op"] == "decode":
        T, H, K = case["tokens"], case["heads"], case["topk"]
        seen = T * K if not case["ragged"] else T * K * 0.485 * (T - 1) / T if T > 1 else 0
        rows = seen if case["own_pools"] else min(seen, case["slots"])
        b = rows * ROW + T * (H * (2 * DIM + 2 * LATENT + 4) + 4 * K) + (2 * T * K if case["weights"] else 0)
        return {"bytes": b, "flops": 2 * seen * H * (DIM + LATENT)}
    R, S, Q = case["requests"], case["slots"], case["topk"]
    miss = Q // 4
    per = 12 * S + Q * (4 + 4 + 4 + 1 + 1 + 4 + 2) + miss * (8 + 4 + 8 + 4 + 4)
    return {"bytes": R * per, "flops": 2 * R * S}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _two_to(e):
    """2.0 ** e in 64 bits, exactly (a power function may be off in its last bit)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _values64(rows):
    """Bytes [n, 416] -> values [n, 576] in 64 bits, value by value from the row's definition."""
    i = torch.arange(LATENT, device=rows.device)
    nibble = (i % 8) // 2 + 4 * (i % 2)
    byte = rows[:, (i // 8) * 4 + nibble // 2].long()
    code = torch.where(nibble % 2 == 1, byte // 16, byte % 16)
    b = rows[:, 256 + i // GROUP].long()
    scale = (1.0 + (b % 8).double() / 8.0) * _two_to(b // 8 - BIAS)
    rope = rows[:, 288:].contiguous().view(torch.bfloat16).double()
    return torch.cat([(code - 8).double() * scale, rope], 1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rows":
        x = st["src"].double()
        lat = x[:, :LATENT].reshape(-1, LATENT // GROUP, GROUP)
        top = lat.abs().max(-1).values
        top = top / torch.full_like(top, 7.0)
        _, e = torch.frexp(top.clamp(min=2.0 ** -60))
        step = _two_to(e - 4)  # three bits behind the point of a number in [1, 2)
        s = torch.round(top / step) * step
        s = s.clamp(2.0 ** -BIAS, 15.0 / 8.0 * 2.0 ** (31 - BIAS))
        lat = torch.round(lat / s[..., None]).clamp(-7, 7) * s[..., None]
        return {"rows": torch.cat([lat.reshape(-1, LATENT), x[:, LATENT:]], 1)}
    if case["op"] == "decode":
        q, slots, out, lse, wsum = st["q"].double(), st["slots"], [], [], []
        for t in range(q.shape[0]):
            pool = st["pool"][t] if st["pool"].dim() == 3 else st["pool"]
            live = slots[t] >= 0
            kv = _values64(pool[slots[t][live].long()])
            s = q[t] @ kv.T * SCALE
            a = torch.softmax(s, -1)
            out.append(a @ kv[:, :LATENT])
            lse.append(torch.logsumexp(s, -1))
            w = torch.zeros(slots.shape[1], device=q.device, dtype=torch.float64)
            w[live] = a.sum(0)
            wsum.append(w)
        got = {"out": torch.stack(out), "lse": torch.stack(lse)}
        return got | ({"weights": torch.stack(wsum)} if st["weights"] else {})
    # the first step: no earlier weights, so the scores decay, and those of the evicted slots go to zero
    R, S = st["score"].shape
    score = st["score"].double() * DECAY
    for r in range(R):
        res = st["slot_to_token"][r]
        q = st["query"][0][r].long()
        hits = st["token_to_slot"][r][q]
        may = res >= 0
        may[hits[hits >= 0].long()] = False
        if st["keep_from"] is not None:
            may &= res < st["keep_from"][r]
        ids = may.nonzero()[:, 0]
        n = min(max(0, case["target"] - int(st["free_count"][r])), len(ids))
        # in 32 bits, as the order is defined on the stored scores; equal ones by the lower slot
        kept = (st["score"][r] * DECAY)[ids]
        score[r, ids[kept.sort(stable=True).indices[:n]]] = 0.0
    return {"score": score, "slot": None, "hit": None, "install": None, "evicted": None, "evicted_count": None,
            "token_to_slot": None, "slot_to_token": None, "free_stack": None, "free_count": None}
