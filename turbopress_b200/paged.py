"""Paged key-value cache: append, attention of new tokens, eviction.

``DecodeStep`` owns contiguous caches sized for the longest sequence and steps
one token.  ``PagedKVCache`` is a pool of pages shared by all sequences, steps
any number of tokens per sequence (a prompt's chunk, drafted tokens), and can be
held to a budget of slots by the attention weight each slot has received.

    cache = PagedKVCache(batch=8, kv_heads=8, head_dim=128, num_pages=4096, page_size=16, max_pages=512, layers=36)
    cache.block_table[b, :n] = pages                   # the caller assigns pages
    q = cache.append(rotary, q, k, v, layer=i)         # rotary positions, k and v into the pages
    out = cache.attend(q, layer=i)                     # [batch, tokens, q_heads, head_dim]
    cache.advance(tokens)                              # after the last layer

``lengths`` (slots in use; negative for an idle sequence) and ``next_pos`` (the
next token's position) live on the device, so a step needs no host round trip.
Every call runs on the current stream of the cache's device; one cache serves
one stream at a time (its workspace is shared by its calls).  No gradients are
recorded.
"""

from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from . import _abi
from .rotary import Rotary


class _PagedCache(ctypes.Structure):
    """Mirror of ``tp_paged_cache``."""

    _fields_ = [(nm, ctypes.c_void_p) for nm in ("k_pages", "v_pages", "block_table", "lengths", "scores", "positions")] + [
        (nm, ctypes.c_int64) for nm in ("num_pages", "page_stride", "head_stride", "token_stride", "table_stride")] + [
        (nm, ctypes.c_int32) for nm in ("batch", "kv_heads", "head_dim", "page_size", "max_pages", "dtype")]


class _AttnArgs(ctypes.Structure):
    """Mirror of ``tp_paged_attn_args``."""

    _fields_ = [("q", ctypes.c_void_p), ("out", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("tokens", ctypes.c_int32),
                ("q_heads", ctypes.c_int32), ("softmax_scale", ctypes.c_float), ("accumulate", ctypes.c_int32),
                ("wait_polls", ctypes.c_int32), ("wait_hold", ctypes.c_int32)]


class _WeightsArgs(ctypes.Structure):
    """Mirror of ``tp_paged_weights_args``."""

    _fields_ = [("q", ctypes.c_void_p), ("lse", ctypes.c_void_p), ("counts", ctypes.c_void_p), ("tokens", ctypes.c_int32),
                ("q_heads", ctypes.c_int32), ("softmax_scale", ctypes.c_float), ("reserved", ctypes.c_int32)]


class _EvictArgs(ctypes.Structure):
    """Mirror of ``tp_evict_args``."""

    _fields_ = [("next_pos", ctypes.c_void_p), ("new_lengths", ctypes.c_void_p), ("new_scores", ctypes.c_void_p),
                ("new_positions", ctypes.c_void_p), ("budget", ctypes.c_int32), ("recent", ctypes.c_int32),
                ("sinks", ctypes.c_int32)]


class PagedKVCache:
    """Pages, block table and lengths of a batch of sequences, layer by layer.

    The kernels have the addresses of its tensors: write into them (``copy_``,
    indexing); another tensor in the place of one is refused."""

    _FIXED = frozenset(("k_pages", "v_pages", "block_table", "lengths", "scores", "positions"))

    def __setattr__(self, name: str, value) -> None:
        if name in self._FIXED and self.__dict__.get(name, value) is not value:  # (an in-place operator gives back the same)
            raise AttributeError(f"{name} keeps its tensor: write into it (cache.{name}.copy_(...)), or make another cache "
                                 "with from_tensors")
        object.__setattr__(self, name, value)

    def __init__(self, batch: int, kv_heads: int, head_dim: int, num_pages: int, page_size: int, max_pages: int, *,
                 layers: int = 1, dtype: torch.dtype = torch.float16, track_weights: bool = False, device="cuda") -> None:
        """``track_weights``: keep each slot's accumulated attention weight and
        position, which eviction goes by."""
        dev = torch.device(device)
        pool = (layers, num_pages, kv_heads, page_size, head_dim)
        slots = (layers, batch, kv_heads, max_pages * page_size)
        self._setup(torch.zeros(pool, dtype=dtype, device=dev), torch.zeros(pool, dtype=dtype, device=dev),
                    torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev),
                    torch.zeros(batch, dtype=torch.int32, device=dev),
                    torch.zeros(slots, dtype=torch.float32, device=dev) if track_weights else None,
                    torch.full(slots, -1, dtype=torch.int32, device=dev) if track_weights else None, None)

    @classmethod
    def from_tensors(cls, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, lengths: Tensor, *,
                     scores: Tensor | None = None, positions: Tensor | None = None,
                     next_pos: Tensor | None = None) -> "PagedKVCache":
        """Over a program's own tensors, shared and not copied: pages
        [num_pages, kv_heads, page_size, head_dim] (any strides with contiguous
        elements, so ``x.transpose(1, 2)`` of token-major pages too) or with a
        leading axis of layers, block_table int32 [batch, max_pages], lengths
        int32 [batch], scores fp32 and positions int32 [(layers,) batch,
        kv_heads, max_pages * page_size], next_pos int32 [batch] (default: a
        copy of lengths)."""
        self = cls.__new__(cls)
        if k_pages.dim() == 4:
            k_pages, v_pages = k_pages[None], v_pages[None]
            scores = None if scores is None else scores[None]
            positions = None if positions is None else positions[None]
        self._setup(k_pages, v_pages, block_table, lengths, scores, positions, next_pos)
        return self

    def _setup(self, k_pages: Tensor, v_pages: Tensor, block_table: Tensor, lengths: Tensor, scores: Tensor | None,
               positions: Tensor | None, next_pos: Tensor | None) -> None:
        if k_pages.dim() != 5 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
            raise ValueError("k_pages and v_pages must share the shape [(layers,) num_pages, kv_heads, page_size, head_dim] "
                             "and the dtype")
        dev = _abi.require_cuda(k_pages, v_pages, block_table, lengths, scores, positions, next_pos)
        L, self.num_pages, self.kv_heads, self.page_size, self.head_dim = k_pages.shape
        if k_pages.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"pages must be fp16 or bf16, got {k_pages.dtype}")
        if k_pages.stride(4) != 1 or v_pages.stride() != k_pages.stride():
            raise ValueError("page elements must be contiguous, and k_pages and v_pages share their strides")
        if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.stride(1) != 1:
            raise ValueError("block_table must be int32 [batch, max_pages] with contiguous rows")
        self.batch, self.max_pages = block_table.shape
        self.capacity = self.max_pages * self.page_size
        for t, nm in ((lengths, "lengths"), (next_pos, "next_pos")):
            if t is not None and (t.shape != (self.batch,) or t.dtype != torch.int32 or not t.is_contiguous()):
                raise ValueError(f"{nm} must be contiguous int32 [batch]")
        slots = (L, self.batch, self.kv_heads, self.capacity)
        for t, dt, nm in ((scores, torch.float32, "scores"), (positions, torch.int32, "positions")):
            if t is not None and (t.shape != slots or t.dtype != dt or not t.is_contiguous()):
                raise ValueError(f"{nm} must be contiguous {dt} {slots}")
        self.device, self.layers, self.dtype = dev, L, k_pages.dtype
        self.k_pages, self.v_pages, self.block_table, self.lengths = k_pages, v_pages, block_table, lengths
        self.scores, self.positions = scores, positions
        self.next_pos = lengths.clone() if next_pos is None else next_pos
        self._structs = [_PagedCache(
            k_pages[i].data_ptr(), v_pages[i].data_ptr(), block_table.data_ptr(), lengths.data_ptr(),
            None if scores is None else scores[i].data_ptr(), None if positions is None else positions[i].data_ptr(),
            self.num_pages, k_pages.stride(1), k_pages.stride(2), k_pages.stride(3), block_table.stride(0), self.batch,
            self.kv_heads, self.head_dim, self.page_size, self.max_pages, _abi.dtype_code(self.dtype)) for i in range(L)]
        self._ws: Tensor | None = None
        self._evict_ws: Tensor | None = None
        self._captured: list[Tensor] = []  # workspaces of attend and of eviction that graphs were recorded with
        self._evict_captured: list[Tensor] = []
        self._plans: dict[tuple, _AttnArgs] = {}
        self._wait = (0, 0)
        self._append_plans: dict[Rotary, dict] = {}
        self._evict_bytes: dict[int, int] = {}
        self._slots = None if scores is None or positions is None else [(scores[i], positions[i]) for i in range(L)]

    def _layer(self, layer: int) -> int:
        """Address of the layer's ``tp_paged_cache``."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"layer {layer} not in [0, {self.layers})")
        return ctypes.addressof(self._structs[layer])

    # -- one step ---------------------------------------------------------------
    def append(self, rotary: Rotary, q: Tensor, k: Tensor, v: Tensor, positions: Tensor | None = None, *, layer: int = 0,
               q_norm: Tensor | None = None, k_norm: Tensor | None = None, eps: float = 1e-6,
               inverse: bool = False) -> Tensor:
        """Rotary positions of a step's q [batch, tokens, q_heads, head_dim] and
        k, and the append of k, v [batch, tokens, kv_heads, head_dim] behind
        ``lengths``; returns the rotated q.  ``positions`` int64 [batch,
        tokens], by default ``next_pos`` onwards.  ``lengths`` stays: call
        ``advance`` once all layers have the step's tokens.  Tokens of idle
        sequences, past the capacity or without a page are not stored."""
        plans = self._append_plans.get(rotary)
        if plans is None:
            if rotary.device != self.device or rotary.head_dim != self.head_dim:
                raise ValueError("the rotary's device and head_dim differ from the cache's")
            if len(self._append_plans) >= 16:  # (a program has one, or one per kind of layer)
                self._append_plans.clear()
            plans = self._append_plans[rotary] = {}
        a, out, keep = rotary._args(plans, self._appendable, q, k, v, positions, q_norm, k_norm, eps, inverse)
        if positions is None:
            a.base = self.next_pos.data_ptr()
        addr = self._layer(layer)
        if a.tokens:
            _abi.launch(_abi.lib().tp_rotary, "append", self.device.index, ctypes.addressof(a), addr)
        return out

    def _appendable(self, plan, q: Tensor, k: Tensor, v: Tensor) -> None:
        """The cache's part of an append's checks; the tokens per sequence."""
        if q.dim() != 4 or q.shape[0] != self.batch or k.shape[-2] != self.kv_heads or q.dtype != self.dtype:
            raise ValueError(f"expected q [{self.batch}, tokens, heads, {self.head_dim}] and k, v with {self.kv_heads} heads, "
                             f"all {self.dtype}")
        plan.seq = max(1, q.shape[1])

    def advance(self, tokens: int | Tensor) -> None:
        """Count ``tokens`` (a number, or int32 [batch]) as cached: after the
        last layer's ``append``.  Idle sequences stay idle.  Fewer than were
        appended drops the last ones (rejected drafts; ``add_weights`` for
        their part in the accumulated weights)."""
        live = (self.lengths >= 0).int() * tokens
        self.lengths.add_(live)
        self.next_pos.add_(live)

    def attend(self, q: Tensor, *, layer: int = 0, scale: float | None = None, accumulate: bool = False,
               return_lse: bool = False):
        """Attention of a step's q [batch, tokens, q_heads, head_dim], already
        appended: token j sees the slots below ``lengths`` and the step's own
        tokens up to itself.  ``scale`` defaults to head_dim ** -0.5.
        ``accumulate`` adds each slot's attention weight to ``scores`` (for
        tokens that may be dropped again: ``add_weights``).  A row that sees nothing (an idle sequence) gives zeros.  Returns out in q's
        shape, with the fp32 log-sum-exp [batch, tokens, q_heads] on request."""
        key = (_abi.meta(q), scale, accumulate)
        plan = self._plans.get(key)
        if plan is None:
            plan = self._checked(q, scale, accumulate)
            if len(self._plans) >= 256:
                self._plans.clear()
            self._plans[key] = plan
        addr = self._layer(layer)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
        if plan.tokens:
            q = q.contiguous()
            a = _AttnArgs.from_buffer_copy(plan)
            a.q, a.out = q.data_ptr(), out.data_ptr()
            if lse is not None:
                a.lse = lse.data_ptr()
            st = _abi.launch(_abi.lib().tp_paged_attn, "attend", self.device.index, ctypes.addressof(a), addr, self._ws.data_ptr(),
                             self._ws.numel())
            if st and _abi.capturing(self.device.index):
                self._keep(self._captured, self._ws)
        return (out, lse) if return_lse else out

    def _checked(self, q: Tensor, scale: float | None, accumulate: bool) -> _AttnArgs:
        """Checks an ``attend`` call by what its key holds; grows the workspace
        (zero-filled) to its sizes."""
        if q.dim() != 4 or q.shape[0] != self.batch or q.shape[3] != self.head_dim:
            raise ValueError(f"expected q [{self.batch}, tokens, heads, {self.head_dim}], got {tuple(q.shape)}")
        if q.dtype != self.dtype or q.device != self.device:
            raise ValueError("q and the pages must share one dtype and device")
        if accumulate and self.scores is None:
            raise ValueError("the cache keeps no scores to accumulate in")
        tokens, heads = q.shape[1], q.shape[2]
        template = _AttnArgs(tokens=tokens, q_heads=heads, softmax_scale=self.head_dim ** -0.5 if scale is None else scale,
                             accumulate=accumulate, wait_polls=self._wait[0], wait_hold=self._wait[1])
        if tokens == 0:
            return template
        need = _abi.lib().tp_paged_attn_workspace_bytes(ctypes.addressof(self._structs[0]), tokens, heads, accumulate)
        if need < 0:
            _abi.check(-need, "attend")
        self._ws = self._grown(self._ws, need)
        return template

    def add_weights(self, q: Tensor, lse: Tensor, counts: Tensor | None = None, *, layer: int = 0, scale: float | None = None) -> None:
        """What ``attend(q, accumulate=True)`` adds to ``scores``, for the first
        ``counts`` int32 [batch] tokens of each sequence (None: all), from the
        log-sum-exp that ``attend(q, return_lse=True)`` gave: for drafts, once
        it is known how many stand and before ``advance``."""
        if q.dim() != 4 or q.shape[0] != self.batch or q.shape[3] != self.head_dim or q.dtype != self.dtype or q.device != self.device:
            raise ValueError(f"expected q [{self.batch}, tokens, heads, {self.head_dim}] {self.dtype} on {self.device}, got "
                             f"{tuple(q.shape)} {q.dtype} on {q.device}")
        if self.scores is None:
            raise ValueError("the cache keeps no scores to accumulate in")
        if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or lse.device != self.device:
            raise ValueError(f"lse must be float32 {tuple(q.shape[:3])} on {self.device}")
        if counts is not None and (counts.shape != (self.batch,) or counts.dtype != torch.int32 or counts.device != self.device):
            raise ValueError(f"counts must be int32 [{self.batch}] on {self.device}")
        addr = self._layer(layer)
        if not q.shape[1]:
            return
        q, lse = q.contiguous(), lse.contiguous()
        counts = None if counts is None else counts.contiguous()
        a = _WeightsArgs(q.data_ptr(), lse.data_ptr(), _abi.ptr(counts), q.shape[1], q.shape[2],
                         self.head_dim ** -0.5 if scale is None else scale, 0)
        _abi.launch(_abi.lib().tp_paged_weights, "add_weights", self.device.index, ctypes.addressof(a), addr)

    def _grown(self, ws: Tensor | None, need: int) -> Tensor:
        """``ws`` if it holds ``need`` bytes, else a zero-filled one that does."""
        if ws is not None and ws.numel() >= need:
            return ws
        if _abi.capturing(self.device.index):
            raise RuntimeError("the workspace has to grow: run this call once before capturing it")
        if ws is not None:  # the calls so far are on this stream or before it
            ws.record_stream(torch.cuda.current_stream(self.device))
        return torch.zeros(need, dtype=torch.uint8, device=self.device)

    @staticmethod
    def _keep(kept: list[Tensor], ws: Tensor) -> None:
        """A graph that is being recorded uses ``ws``: it stays, also when it is outgrown."""
        if not kept or kept[-1] is not ws:
            kept.append(ws)

    def status(self) -> None:
        """Raise if a device-side wait of an ``attend`` gave up, in a graph's
        replay too (synchronizes)."""
        failed = None
        for ws in {id(w): w for w in (*self._captured, self._ws) if w is not None}.values():
            try:
                _abi.launch(_abi.lib().tp_paged_attn_status, "attend", self.device.index, ws.data_ptr())
            except RuntimeError as e:  # (the others' words are read and cleared as well)
                failed = failed or e
        if failed is not None:
            raise failed

    def set_wait(self, polls: int = 0, hold: int = 0) -> None:
        """Polls after which an ``attend`` gives up waiting for a copy (0: the
        default), and (``hold`` > 0) a copy of tile ``hold - 1`` of each block
        that is never begun, so that the wait runs out.  Used to test that
        path; every other run keeps 0."""
        if polls < 0 or hold < 0 or (hold and not polls):
            raise ValueError("polls and hold must be >= 0, and a hold needs its own polls")
        self._wait = (polls, hold)
        self._plans.clear()

    # -- a bounded cache --------------------------------------------------------
    def evict_slots(self, budget: int, *, recent: int = 0, sinks: int = 0, layer: int = 0) -> tuple[Tensor, Tensor, Tensor]:
        """Keep ``budget`` slots of each sequence that has more, per kv head:
        those of the last ``recent`` positions and of the first ``sinks``, then
        those of largest accumulated weight (the lower slot on equality).  The
        kept slots above the budget move into the freed ones below it, in
        place; returns the layer's new (lengths [batch], scores, positions
        [batch, kv_heads, capacity]).  The cache itself still has the old ones:
        ``evict`` does all layers and takes them over."""
        if self._slots is None:
            raise ValueError("eviction needs a cache with scores and positions")
        addr, lib = self._layer(layer), _abi.lib()
        need = self._evict_bytes.get(budget)
        if need is None:
            need = lib.tp_cache_evict_workspace_bytes(addr, budget)
            if need < 0:
                _abi.check(-need, "evict")
            self._evict_ws = self._grown(self._evict_ws, need)
            self._evict_bytes[budget] = need
        scores, positions = self._slots[layer]
        new = (torch.empty_like(self.lengths), torch.empty_like(scores), torch.empty_like(positions))
        a = _EvictArgs(self.next_pos.data_ptr(), new[0].data_ptr(), new[1].data_ptr(), new[2].data_ptr(), budget, recent, sinks)
        st = _abi.launch(lib.tp_cache_evict, "evict", self.device.index, ctypes.addressof(a), addr, self._evict_ws.data_ptr(),
                         self._evict_ws.numel())
        if st and _abi.capturing(self.device.index):
            self._keep(self._evict_captured, self._evict_ws)
        return new

    def evict(self, budget: int, *, recent: int = 0, sinks: int = 0) -> None:
        """``evict_slots`` of every layer; ``lengths``, ``scores`` and
        ``positions`` are then those of the kept slots.  ``next_pos`` stays, so
        later tokens keep their true positions."""
        kept = [self.evict_slots(budget, recent=recent, sinks=sinks, layer=i) for i in range(self.layers)]
        for i, (_, scores, positions) in enumerate(kept):
            self.scores[i].copy_(scores)
            self.positions[i].copy_(positions)
        self.lengths.copy_(kept[0][0])
