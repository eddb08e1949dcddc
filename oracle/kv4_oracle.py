"""CPU restatement of the 4-bit MLA cache and of the attention-weight slot pools (test infrastructure).

Everything is written from the definitions, in 64 bits and one value or one slot at a time where
the order matters.  The reference project has no counterpart of these operators.
"""

from __future__ import annotations

import numpy as np

LATENT, ROPE, GROUP, ROW = 512, 64, 16, 416
BIAS = 18


def bf16_round(x: np.ndarray) -> np.ndarray:
    """Nearest bf16 (ties to even) of finite 32-bit values, as 32-bit floats."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    b = (b + 0x7FFF + ((b >> 16) & 1)) >> 16 << 16
    return b.astype(np.uint32).view(np.float32)


def scale_of(byte: np.ndarray) -> np.ndarray:
    b = np.asarray(byte).astype(np.int64)
    return np.ldexp(1.0 + (b % 8) / 8.0, b // 8 - BIAS)


def nearest_scale(a: float) -> int:
    """The scale byte nearest to a / 7 (ties to the even byte), a >= 0, by comparing with every byte's value."""
    s = scale_of(np.arange(256)) * 7.0  # exact in 64 bits, like 16-bit inputs' maxima
    hi = int(np.searchsorted(s, a))
    if hi == 0:
        return 0
    if hi == 256:
        return 255
    lo = hi - 1
    mid = s[lo] + s[hi]
    if 2 * a == mid:
        return lo if lo % 2 == 0 else hi
    return hi if 2 * a > mid else lo


def pack(rows: np.ndarray) -> np.ndarray:
    """[n, 576] values (of a 16-bit type, as floats) -> [n, 416] bytes."""
    rows = np.asarray(rows, np.float64)
    out = np.zeros((rows.shape[0], ROW), np.uint8)
    for i, row in enumerate(rows):
        for g in range(LATENT // GROUP):
            x = row[g * GROUP: (g + 1) * GROUP]
            byte = nearest_scale(float(np.abs(x).max()))
            out[i, 256 + g] = byte
            s = float(scale_of(byte))
            n = np.clip(np.rint(x / s), -7, 7).astype(np.int64) + 8  # x / s: a tie is exact in 64 bits
            for k in range(GROUP):
                v = g * GROUP + k
                nibble = (v % 8) // 2 + 4 * (v % 2)
                out[i, (v // 8) * 4 + nibble // 2] |= np.uint8(n[k] << (4 * (nibble % 2)))
        rope = bf16_round(row[LATENT:].astype(np.float32)).view(np.uint32) >> 16
        out[i, 288:] = rope.astype(np.uint16).view(np.uint8)
    return out


def unpack(b: np.ndarray) -> np.ndarray:
    """[n, 416] bytes -> [n, 576] values in 64 bits."""
    v = np.arange(LATENT)
    nibble = (v % 8) // 2 + 4 * (v % 2)
    code = (b[:, (v // 8) * 4 + nibble // 2] >> (4 * (nibble % 2)).astype(np.uint8)) & 15
    lat = (code.astype(np.float64) - 8.0) * scale_of(b[:, 256 + v // GROUP])
    rope = (np.ascontiguousarray(b[:, 288:]).view(np.uint16).astype(np.uint32) << 16).view(np.float32)
    return np.concatenate([lat, rope.astype(np.float64)], 1)


def attention(q: np.ndarray, pool: np.ndarray, slots: np.ndarray, scale: float):
    """One token: q [heads, 576], pool [rows, 416] bytes, slots [topk] (-1: not there).

    Returns out [heads, 512], lse [heads], weights [topk], and the magnitudes the error bounds are made
    of: mag [heads, 512] = sum p |v|, smag [heads] = max over entries of scale * sum |q| |k|."""
    q = np.asarray(q, np.float64)
    live = (slots >= 0) & (slots < pool.shape[0])
    H = q.shape[0]
    if not live.any():
        return (np.zeros((H, LATENT)), np.full(H, -np.inf), np.zeros(len(slots)), np.zeros((H, LATENT)), np.zeros(H))
    kv = unpack(pool[slots[live]])
    s = q @ kv.T * scale
    m = s.max(1, keepdims=True)
    e = np.exp(s - m)
    total = e.sum(1, keepdims=True)
    p = e / total
    w = np.zeros(len(slots))
    w[live] = p.sum(0)
    return (p @ kv[:, :LATENT], (m + np.log(total))[:, 0], w, p @ np.abs(kv[:, :LATENT]),
            (np.abs(q) @ np.abs(kv).T * scale).max(1))


class WeightPool:
    """One request's slots, evicted by accumulated weight; serial, slot by slot."""

    def __init__(self, slots: int, target: int, decay: float):
        self.S, self.target, self.decay = slots, min(target, slots), np.float32(decay)
        self.key_slot: dict[int, int] = {}
        self.slot_key = [-1] * slots
        self.score = np.zeros(slots, np.float32)
        self.stack = list(range(slots - 1, -1, -1))

    def step(self, query, last_slot=(), last_weight=(), keep_from=2**31 - 1, key_space=2**31 - 1):
        self.score = (self.score * self.decay).astype(np.float32)
        for s, w in zip(last_slot, last_weight):
            w = np.float32(w)
            if 0 <= s < self.S and self.slot_key[s] >= 0 and w >= 0 and np.isfinite(w):
                self.score[s] = np.float32(self.score[s] + w)
        asked = {self.key_slot[k] for k in query if k in self.key_slot}
        may = [s for s in range(self.S) if self.slot_key[s] >= 0 and s not in asked and self.slot_key[s] < keep_from]
        n = min(max(0, self.target - len(self.stack)), len(may))
        gone = sorted(sorted(may, key=lambda s: (self.score[s], s))[:n])
        evicted = []
        for s in gone:
            evicted.append(self.slot_key[s])
            del self.key_slot[self.slot_key[s]]
            self.slot_key[s] = -1
            self.score[s] = 0
            self.stack.append(s)
        slot, hit, install = [], [], []
        for k in query:
            if not 0 <= k < key_space:
                slot.append(-1), hit.append(False), install.append(False)
            elif k in self.key_slot:
                slot.append(self.key_slot[k]), hit.append(True), install.append(False)
            elif self.stack:
                s = self.stack.pop()
                self.key_slot[k], self.slot_key[s] = s, k
                slot.append(s), hit.append(False), install.append(True)
            else:
                slot.append(-1), hit.append(False), install.append(False)
        return slot, hit, install, evicted
