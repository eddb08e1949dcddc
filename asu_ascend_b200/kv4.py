"""The 4-bit MLA cache: 416-byte rows, and sparse attention over the rows that slots name.

A row holds one token's 512 latent values in 4 bits (scales of 8 bits for 16 values each) and its 64
position-encoded values in bf16, in 416 bytes instead of 1152 (bf16) or 656 (fp8): the managed pool,
the host pool and the swap-in over the host link all shrink alike.  To every other part of the package a
row is raw bytes: ``torch.uint8`` pools of ``[rows, 416]`` go through ``HostRowPool.swapin``,
``HostKVStore.write_back``, the managers and ``sparse_mla.resolve_topk`` as they are.

    kv4.pack_rows(latents, pool, slots)              # the cache's write side
    got = kv4.sparse_decode(q, pool, slots, scale)   # got.out, got.lse
    got = kv4.sparse_decode(q, pool, slots, scale, weights=True)
    pools.step(next_topk, slots, got.weights)        # weight_pools: evict what attention does not look at

All calls are asynchronous on the current stream.  With ``ops.set_status_checks(True)`` each call
synchronises and raises on a device status.  Forward only: an input that requires a gradient is refused.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import ops  # noqa: F401  (registers torch.ops.asu.kv4_*)

LATENT, ROPE, GROUP, ROW_BYTES = 512, 64, 16, 416
MAX_HEADS, MAX_TOKENS, MAX_TOPK = 128, 65535, 16384


class KV4Decode(NamedTuple):
    out: torch.Tensor             # [tokens, heads, 512] bf16
    lse: torch.Tensor             # [tokens, heads] fp32, -inf for a token without any entry
    weights: torch.Tensor | None  # [tokens, topk] bf16: each entry's softmax weight, summed over the heads


def new_pool(*rows: int, device: torch.device | str = "cuda") -> torch.Tensor:
    """A zeroed pool of 4-bit rows: ``new_pool(slots)`` or ``new_pool(requests, slots)``.  (A zero row
    stands for very small values, not for zeros: it is meant to be written before it is read.)"""
    return torch.zeros((*rows, ROW_BYTES), dtype=torch.uint8, device=device)


def pack_rows(src: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor | None = None) -> torch.Tensor:
    """``pool[slots[i]] = src[i]`` in 4 bits (row i without ``slots``); -1 skips a row.

    src ``[n, 576]`` bf16 or fp16 (rows may be strided), pool ``[rows, 416]`` uint8, slots ``[n]``
    int32, distinct.  Each value ends within half a step of its group's scale, which is the group's
    largest magnitude / 7 in 4 significant bits; the rope part is kept in bf16.  Returns ``pool``."""
    torch.ops.asu.kv4_pack_rows(src, pool, slots)
    return pool


def unpack_rows(pool: torch.Tensor, slots: torch.Tensor | None = None) -> torch.Tensor:
    """The values of ``pool[slots]`` (all rows without ``slots``) as ``[n, 576]`` bf16, exactly; zeros
    for slot -1."""
    return torch.ops.asu.kv4_unpack_rows(pool, slots)


def sparse_decode(q: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor, scale: float,
                  weights: bool = False) -> KV4Decode:
    """Sparse MLA attention of decode tokens over 4-bit rows.

    q ``[tokens, heads, 576]`` bf16 (any token and head strides), 1 to 128 heads; pool ``[rows, 416]``
    shared by all tokens or ``[tokens, rows, 416]`` with one pool per token (the slot pools of
    ``LruSlotPools`` / ``WeightSlotPools``); slots ``[tokens, topk]`` int32, -1 for an entry that is
    not there (a shorter context, a shortage).  An entry named twice counts twice.  With ``weights``
    the sum over the heads of each entry's softmax weight is returned too, 0 where there is no entry
    (heads sharded over ranks: add the ranks' weights).  A head with a score that is NaN or +inf has NaN
    for ``out`` and ``lse``, and makes the weights of the token's entries NaN.

    With ``weights`` a call takes up to 256 MiB more of device memory while it runs: two bytes a head (of 16, 32, 64 or
    128) and entry, and calls of more tokens than that holds are done in parts."""
    out, lse, w = torch.ops.asu.kv4_sparse_decode(q, pool, slots, scale, weights)
    return KV4Decode(out, lse, w if weights else None)
