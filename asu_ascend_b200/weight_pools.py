"""Per-request slot pools that evict by accumulated attention weight.

``WeightSlotPools`` is ``lru.LruSlotPools`` with another order of eviction: a slot's score is the sum of
the attention weights its token received, faded by ``decay`` per step, and the slots with the lowest
scores leave first.  A token that attention keeps looking at stays, however long ago it was in a
top-k; one that was read once and ignored goes.  Tokens of the step's own top-k never leave, nor do
tokens at or behind ``keep_from`` (the latest positions).  One launch per step does the last step's
accumulation, the eviction and the resolve.
"""

from __future__ import annotations

import torch

from ._lib import DTYPE_BF16, DTYPE_FP32, LRU_STAT_COLS, ST_SHORTAGE, check, raise_on_status
from .lru import LruStepOutput
from .ops import weight_step

_WEIGHT_DTYPES = {torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_FP32}


class WeightSlotPools:
    """Slot pools of ``req_num`` independent requests.

        pools = WeightSlotPools(128, 131072, 8192, free_target=2048, query_count=2048, decay=0.98)
        out = pools.step(topk)                                   # the first step
        host_pool.swapin(record_addr, topk, out.slot, out.install, kv)
        got = kv4.sparse_decode(q, kv, out.slot, scale, weights=True)
        out = pools.step(next_topk, out.slot, got.weights)       # the next: weights, eviction, resolve
    """

    STAT_NAMES = ("hits", "misses", "installs", "shortages", "evictions")

    def __init__(self, req_num: int, key_space: int, slot_count: int, free_target: int, query_count: int,
                 decay: float = 1.0, device: torch.device | str = "cuda"):
        if req_num <= 0 or key_space <= 0 or slot_count <= 0:
            raise ValueError("req_num, key_space, slot_count, query_count must be positive; free_target >= 0")
        d, i32 = torch.device(device), torch.int32
        if d.type != "cuda":
            raise RuntimeError("WeightSlotPools lives in HBM: device must be CUDA")
        self._adopt(torch.full((req_num, key_space), -1, dtype=i32, device=d),
                    torch.full((req_num, slot_count), -1, dtype=i32, device=d),
                    torch.zeros((req_num, slot_count), dtype=torch.float32, device=d),
                    torch.arange(slot_count - 1, -1, -1, dtype=i32, device=d).repeat(req_num, 1),
                    torch.full((req_num,), slot_count, dtype=i32, device=d), free_target, query_count, decay)

    @classmethod
    def from_state(cls, token_to_slot: torch.Tensor, slot_to_token: torch.Tensor, score: torch.Tensor,
                   free_stack: torch.Tensor, free_count: torch.Tensor, *, free_target: int, query_count: int,
                   decay: float = 1.0) -> "WeightSlotPools":
        """Pools over state tensors that the caller holds (used in place, not copied):
        token_to_slot ``[R, key_space]``, slot_to_token / free_stack ``[R, S]`` and free_count ``[R]``
        int32, score ``[R, S]`` fp32, finite and not negative."""
        self = cls.__new__(cls)
        self._adopt(token_to_slot, slot_to_token, score, free_stack, free_count, free_target, query_count, decay)
        return self

    def _adopt(self, token_to_slot, slot_to_token, score, free_stack, free_count, free_target, query_count,
               decay) -> None:
        if token_to_slot.dim() != 2 or slot_to_token.dim() != 2:
            raise ValueError("token_to_slot must be [R, key_space] and slot_to_token [R, slots]")
        (R, K), S = token_to_slot.shape, slot_to_token.shape[1]
        if R <= 0 or K <= 0 or S <= 0 or query_count <= 0 or free_target < 0:
            raise ValueError("req_num, key_space, slot_count, query_count must be positive; free_target >= 0")
        if S > 16384 or query_count > 4096 or K >= 2**31:
            raise ValueError("supported: slot_count <= 16384, query_count <= 4096, key_space < 2**31")
        if not 0.0 <= decay <= 1.0:
            raise ValueError("decay must be in [0, 1]")
        self.device = token_to_slot.device
        for name, t, shape, dtype in (
                ("token_to_slot", token_to_slot, (R, K), torch.int32),
                ("slot_to_token", slot_to_token, (R, S), torch.int32), ("score", score, (R, S), torch.float32),
                ("free_stack", free_stack, (R, S), torch.int32), ("free_count", free_count, (R,), torch.int32)):
            if tuple(t.shape) != shape or t.dtype != dtype or not t.is_contiguous() or t.device != self.device:
                raise RuntimeError(f"{name} must be a contiguous {dtype} tensor {list(shape)} on {self.device}")
        if self.device.type != "cuda":
            raise RuntimeError("WeightSlotPools lives in HBM: device must be CUDA")
        self.req_num, self.key_space, self.slot_count = R, K, S
        self.free_target, self.query_count, self.decay = min(free_target, S), query_count, float(decay)
        self.token_to_slot, self.slot_to_token, self.score = token_to_slot, slot_to_token, score
        self.free_stack, self.free_count = free_stack, free_count
        self.stats = torch.zeros((R, LRU_STAT_COLS), dtype=torch.int64, device=self.device)
        self.status = torch.zeros((R,), dtype=torch.int32, device=self.device)
        self._out = self.new_output()

    def new_output(self) -> LruStepOutput:
        """Output buffers for one step (step() reuses its own set unless given one)."""
        d, R, Q = self.device, self.req_num, self.query_count
        return LruStepOutput(
            slot=torch.empty((R, Q), dtype=torch.int32, device=d),
            hit=torch.empty((R, Q), dtype=torch.bool, device=d),
            install=torch.empty((R, Q), dtype=torch.bool, device=d),
            evicted=torch.full((R, max(self.free_target, 1)), -1, dtype=torch.int32, device=d),
            evicted_count=torch.zeros((R,), dtype=torch.int32, device=d),
        )

    def step(self, query: torch.Tensor, last_slot: torch.Tensor | None = None,
             last_weight: torch.Tensor | None = None, keep_from: torch.Tensor | None = None,
             out: LruStepOutput | None = None, stream: torch.cuda.Stream | None = None) -> LruStepOutput:
        """Advance every request by one step with ``query`` [R, Q] int32 (CUDA, contiguous).

        ``last_slot`` [R, n] int32 and ``last_weight`` [R, n] bf16 or fp32 are the entries whose weights
        this step accumulates first: usually the last step's ``out.slot`` and the weights that its
        attention returned (-1 slots are not there; n <= 4096).  ``keep_from`` [R] int32: tokens at or
        behind it stay.  ``last_slot`` may be the ``slot`` buffer that this step writes."""
        dev, R = self.device, self.req_num
        if query.dtype != torch.int32 or query.device != dev or not query.is_contiguous():
            raise RuntimeError("query must be a contiguous int32 tensor on the pool's device")
        if query.shape != (R, self.query_count):
            raise RuntimeError(f"query must be [{R}, {self.query_count}], got {tuple(query.shape)}")
        n, wtype, lptr, wptr = 0, DTYPE_FP32, None, None
        if last_slot is not None and last_weight is not None:
            if last_slot.dtype != torch.int32 or last_slot.device != dev or not last_slot.is_contiguous():
                raise RuntimeError("last_slot must be a contiguous int32 tensor on the pool's device")
            wtype = _WEIGHT_DTYPES.get(last_weight.dtype)
            if wtype is None or last_weight.device != dev or not last_weight.is_contiguous():
                raise RuntimeError("last_weight must be a contiguous bfloat16 or float32 tensor on the pool's device")
            shape = last_slot.shape
            if len(shape) != 2 or shape[0] != R or last_weight.shape != shape:
                raise RuntimeError(f"last_slot and last_weight must both be [{R}, n]")
            n, lptr, wptr = shape[1], last_slot.data_ptr(), last_weight.data_ptr()
            if n > 4096:
                raise RuntimeError(f"at most 4096 weights a request, got {n}")
        elif last_slot is not None or last_weight is not None:
            raise RuntimeError("last_slot and last_weight go together")
        if keep_from is not None and (keep_from.dtype != torch.int32 or keep_from.device != dev
                                      or keep_from.shape != (R,) or not keep_from.is_contiguous()):
            raise RuntimeError(f"keep_from must be a contiguous int32 tensor [{R}] on the pool's device")
        o = self._out if out is None else self._checked(out)
        check(weight_step(
            dev.index, stream is not None, None if stream is None else stream.cuda_stream, self.token_to_slot.data_ptr(),
            self.slot_to_token.data_ptr(), self.score.data_ptr(), self.free_stack.data_ptr(), self.free_count.data_ptr(),
            lptr, wptr, wtype, n, self.decay, None if keep_from is None else keep_from.data_ptr(), query.data_ptr(),
            o.slot.data_ptr(), o.hit.data_ptr(), o.install.data_ptr(), o.evicted.data_ptr(), o.evicted.shape[1],
            o.evicted_count.data_ptr(), self.stats.data_ptr(), self.status.data_ptr(), R, self.key_space,
            self.slot_count, self.query_count, self.free_target), "asu_weight_step")
        return o

    def _checked(self, out: LruStepOutput) -> LruStepOutput:
        R, Q = self.req_num, self.query_count
        for name, shape, dtype in (("slot", (R, Q), torch.int32), ("hit", (R, Q), torch.bool), ("install", (R, Q), torch.bool),
                                   ("evicted", None, torch.int32), ("evicted_count", (R,), torch.int32)):
            t = getattr(out, name)
            if name == "evicted":
                shape = (R, max(t.shape[-1], self.free_target, 1))
            if tuple(t.shape) != shape or t.dtype != dtype or t.device != self.device or not t.is_contiguous():
                raise RuntimeError(f"out.{name} must be one of new_output()'s: contiguous {dtype} on the pool's device")
        return out

    def check_status(self, ignore: int = ST_SHORTAGE) -> None:
        raise_on_status(self.status, "asu_weight_step", ignore)

    def totals(self) -> dict:
        return dict(zip(self.STAT_NAMES, self.stats.sum(0).cpu().tolist()))
