"""Cache eviction by accumulated attention weight over the C ABI (section "cache eviction" of include/psi_hip.h): what a
long sequence keeps of its cache.  The reference has no counterpart; its caches grow with their sequences.

  page_weights            the accumulators beside a page arena, f32 [pages][KV heads][tokens per page]
  GQASplitKVSingleQKernels.invoke_attend_weights_bucketed (gqa.py), GQA.record with `GQAInput.kv_weights`
                          decode attention that also accumulates
  GQAKVObserveKernels     accumulates what a prompt's last tokens attend to
  GQAKVEvictionKernels    selects the positions to keep per (request, KV head) and moves them to the front

A request that was compacted holds `budget` tokens: its next token goes to position `budget` of the cache, while its
rotary position counts on.  Tensors are torch tensors (torch is only the allocator); launches go to the device's
stream."""
import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np

from . import _lib as L
from .gqa import Device, Dtype, GQAPageTableLayout, _cfg_struct, _check_page_weights, _is_stored, _tokens_per_page


@dataclass(frozen=True)
class GQAKVEvictionConfig:
    num_q_heads: int
    num_kv_heads: int
    head_dim: int
    scale: float
    page_bytes: int
    page_table_layout: GQAPageTableLayout
    dtype: Dtype

    def struct(self):
        return _cfg_struct(self.num_q_heads, self.num_kv_heads, self.head_dim, self.scale, self.page_bytes, self.dtype)

    def num_tokens_per_page(self) -> int:
        return _tokens_per_page(self.struct())


def page_weights(device: Device, config, num_pages: int):
    """Accumulators for an arena of `num_pages` pages, zeroed; `config` is any of the kernels' configs.

    Only a step that accumulates and an observation (from `num_held` on) start the accumulators of new tokens from zero.
    Where other steps append too (prefill, verify), observe their tokens before the next accumulating step or selection,
    or zero a page's accumulators when it is issued again."""
    import torch

    out, cfg = ctypes.c_uint64(), config.struct()
    L.check(L.load().psi_hip_kv_page_weights_bytes(ctypes.byref(cfg), num_pages, ctypes.byref(out)))
    with torch.cuda.stream(device.stream):
        flat = torch.zeros(out.value // 4, dtype=torch.float32, device=device.torch_device)
    return flat.view(num_pages, cfg.num_kv_heads, -1)


def _u32(values):
    a = np.ascontiguousarray(values)
    if a.size and (a.min() < 0 or a.max() > 0xFFFFFFFF):
        raise ValueError("request slots, positions and counts are unsigned 32-bit numbers")
    return np.ascontiguousarray(a, dtype=np.uint32)


def _p(a):
    return a.ctypes.data_as(ctypes.POINTER(ctypes.c_uint32)) if a is not None else None


# What a launch call passes is made with as little as can be: the smallest launches take less time than ten conversions.
def _addr(t):
    return t.data_ptr() if t is not None else None


def _size(t):
    return t.nbytes if t is not None else 0


def _upload(device: Device, array: np.ndarray):
    import torch

    with torch.cuda.stream(device.stream):
        return torch.from_numpy(array.view(np.int32)).to(device.torch_device)


@dataclass
class GQAKVObservePlan:
    """One batch's windows and rows on the device, with the scratch of its launches: one use at a time."""
    windows: object
    rows: object
    num_windows: int
    num_rows: int
    num_q_tokens: int
    max_window: int
    scratch: object
    max_window_rows: int = 0  # rows of the window that has most; 0: not known


class GQAKVObserveKernels:
    def __init__(self, device: Device, config: GQAKVEvictionConfig):
        config.num_tokens_per_page()  # validates
        self.device, self.config = device, config
        self._cfg, self._layout = config.struct(), config.page_table_layout.struct()
        self._refs = ctypes.byref(self._cfg), ctypes.byref(self._layout)
        self._torch_dtype = config.dtype.torch()

    def prepare(self, req_slots: Sequence[int], token_indices: Sequence[int], cu_tokens: Sequence[int],
                num_held: Optional[Sequence[int]] = None) -> GQAKVObservePlan:
        """`token_indices[r]`: position of request r's first observing token, `cu_tokens` the prefix sums of their
        numbers; `num_held[r]`: positions whose accumulators count already (None: `token_indices`; 0 for a prompt's
        first observation).  psi_hip_kv_observe_plan and one upload."""
        import torch

        rs, ti, cu = _u32(req_slots), _u32(token_indices), _u32(cu_tokens)
        held = _u32(num_held) if num_held is not None else None
        if len(ti) != len(rs) or len(cu) != len(rs) + 1 or (held is not None and len(held) != len(rs)):
            raise ValueError("req_slots, token_indices and num_held name the same requests, cu_tokens one more")
        capacity = 512 + len(rs)
        words = np.empty(8 * len(rs) + 3 * capacity, np.uint32)
        n, most, scratch = ctypes.c_uint32(), ctypes.c_uint32(), ctypes.c_uint64()
        L.check(L.load().psi_hip_kv_observe_plan(
            ctypes.byref(self._cfg), ctypes.byref(self._layout), _p(rs), _p(ti), _p(cu), _p(held), len(rs), _p(words),
            _p(words[8 * len(rs):]), capacity, ctypes.byref(n), ctypes.byref(most), ctypes.byref(scratch)))
        table = _upload(self.device, words[:8 * len(rs) + 3 * n.value])
        with torch.cuda.stream(self.device.stream):
            buffer = torch.empty(scratch.value, dtype=torch.uint8, device=self.device.torch_device)
        bounds = words[:8 * len(rs)].reshape(-1, 8)
        return GQAKVObservePlan(table[:8 * len(rs)], table[8 * len(rs):], len(rs), n.value, int(cu[-1]), most.value,
                                buffer, int((bounds[:, 6] - bounds[:, 5]).max()))

    def invoke(self, plan: GQAKVObservePlan, q, kv_pages, page_ids, page_weights, page_table_index: int,
               decay: float = 1.0):
        """Adds the windows' weights to `page_weights`; `q`: [query tokens][Q heads][head_dim], rotated."""
        _check_page_weights(page_weights, self.device)
        if (q.numel() < plan.num_q_tokens * self.config.num_q_heads * self.config.head_dim or
                q.element_size() != self.config.dtype.item_size() or not _is_stored(q, self._torch_dtype, self.device)):
            raise ValueError("q: contiguous rows of the cache's type on the kernels' device are wanted, one for every "
                             "planned query token")
        if not _is_stored(kv_pages, self._torch_dtype, self.device):
            raise ValueError("kv_pages: a contiguous arena of the configured type on the kernels' device is wanted")
        if plan.scratch.device != self.device.torch_device:
            raise ValueError("plan: one prepared on the kernels' device is wanted")
        L.check(self.device.lib.psi_hip_kv_observe_weights_rows(
            self.device.ctx, *self._refs, _addr(q), plan.num_q_tokens, _addr(kv_pages), _size(kv_pages), _addr(page_ids),
            _addr(plan.windows), plan.num_windows, plan.max_window, _addr(plan.rows), plan.num_rows, plan.max_window_rows,
            _addr(plan.scratch), _size(plan.scratch), _addr(page_weights), _size(page_weights), decay, page_table_index))


@dataclass
class GQAKVEvictionPlan:
    """The requests of an eviction on the device, room for what they keep and the selection's scratch: one use at a
    time."""
    requests: object
    num_reqs: int
    max_cached: int
    kept: object
    scratch: object  # of a selection; None when it needs none


class GQAKVEvictionKernels:
    """Per (request, KV head): the first `num_first` tokens, the last `num_recent`, and the heaviest others up to
    `budget`."""

    def __init__(self, device: Device, config: GQAKVEvictionConfig, budget: int, num_first: int = 0,
                 num_recent: int = 0):
        config.num_tokens_per_page()  # validates
        if budget <= 0 or num_first < 0 or num_recent < 0 or num_first + num_recent > budget:
            raise ValueError("eviction keeps 0 <= num_first + num_recent <= budget tokens, budget positive")
        self.device, self.config = device, config
        self.budget, self.num_first, self.num_recent = budget, num_first, num_recent
        self._cfg, self._layout = config.struct(), config.page_table_layout.struct()
        self._refs = ctypes.byref(self._cfg), ctypes.byref(self._layout)
        self._torch_dtype = config.dtype.torch()

    def prepare(self, req_slots: Sequence[int], num_cached: Sequence[int]) -> GQAKVEvictionPlan:
        """`num_cached[r]`: the tokens that request r's cache holds.  psi_hip_kv_evict_plan and one upload."""
        import torch

        rs, nc = _u32(req_slots), _u32(num_cached)
        if len(rs) != len(nc):
            raise ValueError("req_slots and num_cached name the same requests")
        requests, most = np.empty(2 * len(rs), np.uint32), ctypes.c_uint32()
        L.check(L.load().psi_hip_kv_evict_plan(ctypes.byref(self._cfg), ctypes.byref(self._layout), _p(rs), _p(nc),
                                               len(rs), _p(requests), ctypes.byref(most)))
        scratch = ctypes.c_uint64()
        L.check(L.load().psi_hip_kv_select_scratch_bytes(ctypes.byref(self._cfg), len(rs), most.value,
                                                         ctypes.byref(scratch)))
        with torch.cuda.stream(self.device.stream):
            kept = torch.empty((len(rs), self.config.num_kv_heads, self.budget), dtype=torch.int32,
                               device=self.device.torch_device)
            buffer = (torch.empty(scratch.value, dtype=torch.uint8, device=self.device.torch_device) if scratch.value
                      else None)
        return GQAKVEvictionPlan(_upload(self.device, requests), len(rs), most.value, kept, buffer)

    def _check_plan(self, plan: GQAKVEvictionPlan):
        """A plan has room for what its own kernels keep: another budget or head count would leave it."""
        kept, wanted = plan.kept, (plan.num_reqs, self.config.num_kv_heads, self.budget)
        if kept.shape != wanted or kept.device != self.device.torch_device:
            raise ValueError(f"plan: one prepared by kernels of this budget, head count and device is wanted; it keeps "
                             f"{tuple(plan.kept.shape)} positions on {plan.kept.device}, these kernels {wanted}")

    def invoke_select(self, plan: GQAKVEvictionPlan, page_weights, page_ids, page_table_index: int):
        """The positions to keep, int32 [requests][KV heads][budget], ascending and padded with -1 (the 32-bit
        sentinel); `plan.kept`, which the plan's next selection writes again.  `plan` is one of these kernels' own, or of
        others with the same budget, head count and page table layout."""
        self._check_plan(plan)
        _check_page_weights(page_weights, self.device)
        L.check(self.device.lib.psi_hip_kv_select_kept(
            self.device.ctx, *self._refs, _addr(page_weights), _size(page_weights), _addr(page_ids), _addr(plan.requests),
            plan.num_reqs, plan.max_cached, self.budget, self.num_first, self.num_recent, _addr(plan.kept),
            _addr(plan.scratch), _size(plan.scratch), page_table_index))
        return plan.kept

    def invoke_compact(self, plan: GQAKVEvictionPlan, kept, kv_pages, page_weights, page_ids, page_table_index: int):
        """Moves the kept lines of `kv_pages` and their accumulators (`page_weights` may be None) to the front."""
        self._check_plan(plan)
        if page_weights is not None:
            _check_page_weights(page_weights, self.device)
        if kept is not plan.kept and (kept.dtype != plan.kept.dtype or not kept.is_contiguous() or
                                      kept.numel() != plan.kept.numel() or kept.device != self.device.torch_device):
            raise ValueError("kept: the contiguous int32 [requests][KV heads][budget] of a selection is wanted")
        if not _is_stored(kv_pages, self._torch_dtype, self.device):
            raise ValueError("kv_pages: a contiguous arena of the configured type on the kernels' device is wanted")
        L.check(self.device.lib.psi_hip_kv_compact(
            self.device.ctx, *self._refs, _addr(kv_pages), _size(kv_pages), _addr(page_weights), _size(page_weights),
            _addr(page_ids), _addr(plan.requests), plan.num_reqs, plan.max_cached, self.budget, _addr(kept),
            page_table_index))
