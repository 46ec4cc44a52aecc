"""Batched decode over a paged KV pool (torch device buffers + libkvcache.so).

The reference keeps one sequence in an unpaged pool and "batches" with a
sequential Python loop (src/inference.py:435-447).  This module is the batched
form of the same path: many sequences share one pool of fixed-size pages,
addressed through int32 block tables, and one decode step per layer appends the
new K/V row of every sequence and attends over its whole cached context
(the per-token append of attention.hip:410-415 and the attention of
attention.hip:35-123, for a batch).

Buffers are torch CUDA tensors; work is enqueued on torch's current stream
unless a stream is given.  KV-head sharding across GPUs is a matter of
building each rank's pool with its own ``num_kv_heads`` slice (see
``shard_heads``).
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

import kvcache_ffi as ffi

_TORCH_CODE = {torch.float16: ffi.DTYPE_F16, torch.bfloat16: ffi.DTYPE_BF16,
               torch.float32: ffi.DTYPE_F32}


def _sp(stream) -> Optional[int]:
    s = stream if stream is not None else torch.cuda.current_stream()
    return int(s.cuda_stream) or None


def _i32(t: torch.Tensor) -> int:
    if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous():
        raise ValueError("block tables / rows / positions must be contiguous int32 CUDA tensors")
    return int(t.data_ptr())


def _dev(t: torch.Tensor, name: str, dtype: torch.dtype, numel: int) -> int:
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} CUDA tensor")
    if t.numel() < numel:
        raise ValueError(f"{name} buffer is smaller than expected dimensions.")
    return int(t.data_ptr())


# The operators below run in a few microseconds: their checks look at a tensor as seldom
# as they can, and put a message together only when one fails.
def _on(t: torch.Tensor, name: str, dtype: torch.dtype, numel: int, device: int) -> int:
    """Address of a contiguous tensor of `dtype` on CUDA device `device`, `numel` or larger."""
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous():
        if t.is_cuda and t.get_device() != device:
            raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")
        raise ValueError(f"{name} must be a contiguous {dtype} CUDA tensor")
    if numel and t.numel() < numel:
        raise ValueError(f"{name} buffer is smaller than expected dimensions.")
    return t.data_ptr()


def _token_rows(t: torch.Tensor, name: str, dtype: torch.dtype, shape, device: int):
    """(address, elements between tokens) of (n, heads, dim) rows whose heads are packed."""
    if t.dtype is not dtype or t.get_device() != device:
        raise ValueError(f"{name} must be a {dtype} tensor on cuda:{device}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
    n, heads, dim = shape
    s0, s1, s2 = t.stride()
    if (s2 != 1 and dim > 1) or (s1 != dim and heads > 1) or (s0 < heads * dim and n > 1):
        raise ValueError(f"the heads of a token of {name} must be packed")
    if s0 >= 1 << 31 and n > 1:     # (the call takes it in 32 bits)
        raise ValueError(f"the tokens of {name} are 2^31 elements apart or more")
    return t.data_ptr(), (s0 if n > 1 else heads * dim)


def _counts(a, name: str) -> np.ndarray:
    """Whole numbers as int32, none of them cut to fit."""
    wide = np.asarray(a, dtype=np.int64)
    got = np.ascontiguousarray(wide.astype(np.int32))
    if not np.array_equal(got, wide):
        raise ValueError(f"{name} must fit 32 bits")
    return got


def _stream_on(stream, device: int) -> Optional[int]:
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device) or None
    return int(stream.cuda_stream) or None


def _made_on(stream, device):
    """What is allocated or uploaded inside belongs to `stream` (None: the current one), so
    that its memory goes to another tensor only behind the kernels enqueued there."""
    if stream is None:
        return contextlib.nullcontext()
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream.cuda_stream), device=device)
    return torch.cuda.stream(stream)


def _upload(a: np.ndarray, dev: torch.device) -> torch.Tensor:
    """A tensor of `a` on `dev`, without waiting for the stream's earlier work."""
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t.pin_memory().to(dev, non_blocking=True) if dev.type == "cuda" else t


@dataclass
class PlanInfo:
    n_queries: int
    n_items: int
    n_ctas: int
    scratch_bytes: int


class DecodePlan:
    """Split-K work list for one batch of queries (see kvc_plan_decode)."""

    def __init__(self):
        h = ctypes.c_void_p()
        ffi.check(ffi.lib.kvc_plan_create(ctypes.byref(h)))
        self.handle = h
        self.n_queries = 0
        self.num_heads = 0
        self.ctx_lens: Optional[np.ndarray] = None
        self.flags = 0

    def _set_flag(self, flag: int, on: bool) -> None:
        flags = (self.flags | flag) if on else (self.flags & ~flag)
        ffi.check(ffi.lib.kvc_plan_set_flags(self.handle, flags))
        self.flags = flags

    def set_kv_stable(self, stable: bool = True) -> None:
        """Declare that block tables and KV pages are not written by the kernel
        launched right before each decode (lets the kernel start streaming KV
        early; see KVC_PLAN_KV_STABLE)."""
        self._set_flag(ffi.PLAN_KV_STABLE, stable)

    def set_graph_stable(self, on: bool = True) -> None:
        """Let decode launches of this plan be captured in a CUDA graph and replayed
        after rebuilds for grown contexts (KVC_PLAN_GRAPH); re-capture whenever
        ``generation`` changes.  Set before the first build."""
        self._set_flag(ffi.PLAN_GRAPH, on)

    @property
    def generation(self) -> int:
        """Layout generation: launches captured under another value are stale."""
        g = ctypes.c_uint64()
        ffi.check(ffi.lib.kvc_plan_generation(self.handle, ctypes.byref(g)))
        return g.value

    def info(self) -> PlanInfo:
        n_items, n_ctas = ctypes.c_int(), ctypes.c_int()
        scratch = ctypes.c_size_t()
        ffi.check(ffi.lib.kvc_plan_info(self.handle, ctypes.byref(n_items), ctypes.byref(n_ctas),
                                        ctypes.byref(scratch)))
        return PlanInfo(self.n_queries, n_items.value, n_ctas.value, scratch.value)

    def close(self):
        if self.handle is not None:
            ffi.check(ffi.lib.kvc_plan_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class TreePlan:
    """Work list of one verification step of drafted tokens (see kvc_plan_tree)."""

    def __init__(self):
        h = ctypes.c_void_p()
        ffi.check(ffi.lib.kvc_tree_plan_create(ctypes.byref(h)))
        self.handle = h
        self.n_tokens = 0
        self.num_heads = 0
        self.max_row = 0
        self.ctx_lens: Optional[np.ndarray] = None
        self.node_counts: Optional[np.ndarray] = None

    def info(self) -> PlanInfo:
        n, ctas, scratch = ctypes.c_int(), ctypes.c_int(), ctypes.c_size_t()
        ffi.check(ffi.lib.kvc_tree_plan_info(self.handle, ctypes.byref(n), ctypes.byref(ctas),
                                             ctypes.byref(scratch)))
        return PlanInfo(n.value, ctas.value, ctas.value, scratch.value)

    def close(self):
        if self.handle is not None:
            ffi.check(ffi.lib.kvc_tree_plan_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class PagedKVCache:
    """Paged K/V pool for ``num_layers`` layers on one GPU."""

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int,
                 head_dim: int, dtype: torch.dtype = torch.float16, device: int = 0):
        if dtype not in _TORCH_CODE:
            raise ValueError(f"unsupported KV storage dtype {dtype}")
        h = ctypes.c_void_p()
        ffi.check(ffi.lib.kvc_pool_create(num_layers, num_pages, page_size, num_kv_heads,
                                          head_dim, _TORCH_CODE[dtype], device, ctypes.byref(h)))
        self.handle = h
        self.num_layers = num_layers
        self.num_pages = num_pages
        self.page_size = page_size
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = device

    # -- synthetic contents ------------------------------------------------------
    def fill_normal(self, seed: int, stddev: float = 1.0, layers=None, pages=None, stream=None):
        l0, l1 = layers if layers is not None else (0, self.num_layers)
        p0, p1 = pages if pages is not None else (0, self.num_pages)
        ffi.check(ffi.lib.kvc_pool_fill_normal(self.handle, l0, l1, p0, p1, int(seed),
                                               float(stddev), _sp(stream)))

    def info(self):
        k, v = ctypes.c_void_p(), ctypes.c_void_p()
        lb, phb = ctypes.c_size_t(), ctypes.c_size_t()
        ffi.check(ffi.lib.kvc_pool_info(self.handle, ctypes.byref(k), ctypes.byref(v),
                                        ctypes.byref(lb), ctypes.byref(phb)))
        return {"k": k.value, "v": v.value, "bytes_per_layer": lb.value,
                "bytes_per_page_head": phb.value}

    # -- plan / append / decode ---------------------------------------------------
    def plan(self, ctx_lens: Sequence[int], num_heads: int, rows: Optional[Sequence[int]] = None,
             plan: Optional[DecodePlan] = None, stream=None) -> DecodePlan:
        """Plan attention for query i over positions [0, ctx_lens[i]) of block-table
        row rows[i] (default i)."""
        p = plan if plan is not None else DecodePlan()
        ctx = np.ascontiguousarray(np.asarray(ctx_lens, dtype=np.int32))
        r = None if rows is None else np.ascontiguousarray(np.asarray(rows, dtype=np.int32))
        ffi.check(ffi.lib.kvc_plan_decode(p.handle, self.handle, ffi.np_ptr(r), ffi.np_ptr(ctx),
                                          int(ctx.size), int(num_heads), _sp(stream)))
        p.n_queries = int(ctx.size)
        p.num_heads = int(num_heads)
        p.ctx_lens = ctx
        return p

    def append(self, layer: int, k_new: torch.Tensor, v_new: torch.Tensor,
               block_tables: torch.Tensor, positions: torch.Tensor,
               rows: Optional[torch.Tensor] = None, stream=None):
        n = int(positions.numel())
        row_elems = self.num_kv_heads * self.head_dim
        ffi.check(ffi.lib.kvc_append(
            self.handle, layer, _dev(k_new, "k_new", self.dtype, n * row_elems),
            _dev(v_new, "v_new", self.dtype, n * row_elems), _i32(block_tables),
            int(block_tables.shape[-1]), None if rows is None else _i32(rows), _i32(positions), n,
            _sp(stream)))

    def decode(self, plan: DecodePlan, layer: int, q: torch.Tensor, out: torch.Tensor,
               block_tables: torch.Tensor, scale: float, stream=None):
        n = plan.n_queries * plan.num_heads * self.head_dim
        ffi.check(ffi.lib.kvc_decode(
            self.handle, plan.handle, layer, _dev(q, "q", self.dtype, n),
            _dev(out, "out", self.dtype, n), _i32(block_tables), int(block_tables.shape[-1]),
            float(scale), _sp(stream)))

    def append_decode(self, plan: DecodePlan, layer: int, q: torch.Tensor, k_new: torch.Tensor,
                      v_new: torch.Tensor, out: torch.Tensor, block_tables: torch.Tensor,
                      scale: float, stream=None):
        n = plan.n_queries * plan.num_heads * self.head_dim
        nk = plan.n_queries * self.num_kv_heads * self.head_dim
        ffi.check(ffi.lib.kvc_append_decode(
            self.handle, plan.handle, layer, _dev(q, "q", self.dtype, n),
            _dev(k_new, "k_new", self.dtype, nk), _dev(v_new, "v_new", self.dtype, nk),
            _dev(out, "out", self.dtype, n), _i32(block_tables), int(block_tables.shape[-1]),
            float(scale), _sp(stream)))

    def append_decode_rope(self, plan: DecodePlan, layer: int, q: torch.Tensor,
                           k_new: torch.Tensor, v_new: torch.Tensor, out: torch.Tensor,
                           block_tables: torch.Tensor, scale: float, freq_base: float = 10000.0,
                           neox: bool = False, stream=None):
        """append_decode with q and k_new rotated (RoPE) at each query's position
        first (kvc_append_decode_rope); q and k_new are not modified."""
        n = plan.n_queries * plan.num_heads * self.head_dim
        nk = plan.n_queries * self.num_kv_heads * self.head_dim
        ffi.check(ffi.lib.kvc_append_decode_rope(
            self.handle, plan.handle, layer, _dev(q, "q", self.dtype, n),
            _dev(k_new, "k_new", self.dtype, nk), _dev(v_new, "v_new", self.dtype, nk),
            _dev(out, "out", self.dtype, n), _i32(block_tables), int(block_tables.shape[-1]),
            float(scale), float(freq_base), int(bool(neox)), _sp(stream)))

    def append_decode_xchg(self, plan: DecodePlan, layer: int, q: torch.Tensor,
                           k_new: Optional[torch.Tensor], v_new: Optional[torch.Tensor],
                           xchg_handle, slot: int, total_heads: int, head_offset: int,
                           block_tables: torch.Tensor, scale: float, stream=None):
        """append_decode with the outputs pushed into every rank's exchange slot
        (kvc_append_decode_xchg); see sharding.HeadExchange."""
        n = plan.n_queries * plan.num_heads * self.head_dim
        nk = plan.n_queries * self.num_kv_heads * self.head_dim
        kp = None if k_new is None else _dev(k_new, "k_new", self.dtype, nk)
        vp = None if v_new is None else _dev(v_new, "v_new", self.dtype, nk)
        ffi.check(ffi.lib.kvc_append_decode_xchg(
            self.handle, plan.handle, layer, _dev(q, "q", self.dtype, n), kp, vp, xchg_handle,
            int(slot), int(total_heads), int(head_offset), _i32(block_tables),
            int(block_tables.shape[-1]), float(scale), _sp(stream)))

    def decode_host(self, plan: DecodePlan, layer: int, h_q: torch.Tensor, h_k: torch.Tensor,
                    h_v: torch.Tensor, h_out: torch.Tensor, block_tables: torch.Tensor,
                    scale: float, stream=None):
        """Reference-facing call: host (ideally pinned) buffers in, host result out."""
        for name, t in (("q", h_q), ("k_new", h_k), ("v_new", h_v), ("out", h_out)):
            if t.is_cuda or not t.is_contiguous() or t.dtype != self.dtype:
                raise ValueError(f"{name} must be a contiguous {self.dtype} host tensor")
        ffi.check(ffi.lib.kvc_decode_host(
            self.handle, plan.handle, layer, int(h_q.data_ptr()), int(h_k.data_ptr()),
            int(h_v.data_ptr()), int(h_out.data_ptr()), _i32(block_tables),
            int(block_tables.shape[-1]), float(scale), _sp(stream)))

    def forward_layer(self, plan: DecodePlan, layer: int, x: torch.Tensor, out: torch.Tensor,
                      weights: "DeviceLayerWeights", block_tables: torch.Tensor,
                      eps: float = 1e-5, freq_base: float = 10000.0, neox: bool = False,
                      scale: Optional[float] = None, stream=None):
        """One transformer layer for the plan's queries (kvc_forward_layer_paged):
        x / out (n_queries, hidden) fp16, token i being query i's new token at
        position ctx_i - 1 of its block-table row.  out may be x."""
        n = plan.n_queries * weights.hidden
        sc = default_scale(self.head_dim) if scale is None else float(scale)
        if len(weights.w) != 7 or len(weights.types) != 7:
            raise ValueError("a layer has seven weights: q, k, v, o, gate, up, down")
        for t in weights.w:
            if not t.is_cuda or not t.is_contiguous():
                raise ValueError("weights must be contiguous CUDA tensors")
        w = [int(t.data_ptr()) for t in weights.w]
        ty = [int(t) for t in weights.types]
        ffi.check(ffi.lib.kvc_forward_layer_paged(
            self.handle, plan.handle, layer, _dev(x, "x", torch.float16, n),
            _dev(out, "out", torch.float16, n),
            _dev(weights.attn_norm, "attn_norm", torch.float16, weights.hidden), w[0], ty[0],
            w[1], ty[1], w[2], ty[2], w[3], ty[3],
            _dev(weights.ffn_norm, "ffn_norm", torch.float16, weights.hidden), w[4], ty[4],
            w[5], ty[5], w[6], ty[6], _i32(block_tables), int(block_tables.shape[-1]),
            weights.hidden, weights.intermediate, float(eps), float(freq_base), int(bool(neox)),
            sc, _sp(stream)))

    # -- drafted tokens and beams ---------------------------------------------------
    def append_rope(self, layer: int, q: Optional[torch.Tensor], k_new: torch.Tensor,
                    v_new: torch.Tensor, block_tables: torch.Tensor, positions: torch.Tensor,
                    rows: Optional[torch.Tensor] = None,
                    rope_positions: Optional[torch.Tensor] = None,
                    q_out: Optional[torch.Tensor] = None, freq_base: float = 10000.0,
                    neox: bool = False, stream=None) -> Optional[torch.Tensor]:
        """append with the K rows rotated (RoPE) on the way, and q (n, heads, D) rotated
        into q_out (allocated if not given; returned), in one launch (kvc_append_rope).
        q, k_new, v_new may be slices of one fused projection (n, heads, D): only the
        heads of a token must be packed.  positions are cache slots (negative: padding,
        that token is skipped), rope_positions the angles' positions where they differ."""
        dev, dt, d = self.device, self.dtype, self.head_dim
        n = positions.numel()
        rows_shape = (n, self.num_kv_heads, d)
        kp, ks = _token_rows(k_new, "k_new", dt, rows_shape, dev)
        vp, vs = _token_rows(v_new, "v_new", dt, rows_shape, dev)
        qp = op = None
        heads = qs = 0
        if q is not None:
            if q.dim() != 3:
                raise ValueError("q must be (n, heads, head_dim)")
            heads = q.shape[1]
            qp, qs = _token_rows(q, "q", dt, (n, heads, d), dev)
            if q_out is None:
                with _made_on(stream, dev):
                    q_out = torch.empty((n, heads, d), dtype=dt, device=q.device)
            op = _on(q_out, "q_out", dt, n * heads * d, dev)
        if block_tables.dim() != 2:
            raise ValueError("block_tables must be (rows, pages)")
        ffi.check(ffi.lib.kvc_append_rope(
            self.handle, layer, qp, qs, op, heads, kp, ks, vp, vs,
            _on(block_tables, "block_tables", torch.int32, 0, dev), block_tables.shape[0],
            block_tables.shape[1],
            None if rows is None else _on(rows, "rows", torch.int32, n, dev),
            _on(positions, "positions", torch.int32, n, dev),
            None if rope_positions is None else _on(rope_positions, "rope_positions", torch.int32,
                                                    n, dev),
            n, freq_base, 1 if neox else 0, _stream_on(stream, dev)))
        return q_out

    def plan_tree(self, ctx_lens: Sequence[int], node_counts: Sequence[int], num_heads: int,
                  rows: Optional[Sequence[int]] = None, plan: Optional[TreePlan] = None,
                  stream=None) -> TreePlan:
        """Plan the attention of node_counts[i] drafted tokens per sequence behind
        ctx_lens[i] cached positions of block-table row rows[i] (default i)."""
        ctx, cnt = _counts(ctx_lens, "ctx_lens"), _counts(node_counts, "node_counts")
        r = None if rows is None else _counts(rows, "rows")
        if ctx.shape != cnt.shape or ctx.ndim != 1 or (r is not None and r.shape != ctx.shape):
            raise ValueError("ctx_lens, node_counts and rows must have one entry per sequence")
        p = plan if plan is not None else TreePlan()
        ffi.check(ffi.lib.kvc_plan_tree(p.handle, self.handle, ffi.np_ptr(r), ffi.np_ptr(ctx),
                                        ffi.np_ptr(cnt), ctx.size, int(num_heads),
                                        _stream_on(stream, self.device)))
        p.n_tokens = int(cnt.sum())
        p.num_heads = int(num_heads)
        p.max_row = int(r.max(initial=0)) if r is not None else max(0, ctx.size - 1)
        p.ctx_lens, p.node_counts = ctx, cnt
        return p

    def decode_tree(self, plan: TreePlan, layer: int, q: torch.Tensor,
                    mask: Optional[torch.Tensor], out: torch.Tensor, block_tables: torch.Tensor,
                    scale: float, stream=None):
        """Attention of the plan's drafted tokens (kvc_decode_tree): q, out (tokens,
        heads, D); mask (tokens, words) int32 bit rows (see tree_masks), None for a
        chain.  Their K/V rows must be appended already (append_rope)."""
        dev, dt, t = self.device, self.dtype, plan.n_tokens
        n = t * plan.num_heads * self.head_dim
        mp, words = self._mask(mask, t)
        self._table(block_tables, plan)
        ffi.check(ffi.lib.kvc_decode_tree(
            self.handle, plan.handle, layer, _on(q, "q", dt, n, dev), mp, words,
            _on(out, "out", dt, n, dev), block_tables.data_ptr(), block_tables.shape[1], scale,
            _stream_on(stream, dev)))

    def _mask(self, mask: Optional[torch.Tensor], tokens: int):
        if mask is None:
            return None, 0
        if mask.dim() != 2:
            raise ValueError("mask must be (tokens, words)")
        words = mask.shape[1]
        if words == 0 and tokens:   # (its address is null, which the library takes for a chain)
            raise ValueError("a mask needs at least one word per token")
        return _on(mask, "mask", torch.int32, tokens * words, self.device), words

    def _table(self, block_tables: torch.Tensor, plan: TreePlan) -> None:
        _on(block_tables, "block_tables", torch.int32, 0, self.device)
        if block_tables.dim() != 2:
            raise ValueError("block_tables must be (rows, pages)")
        if plan.n_tokens and plan.max_row >= block_tables.shape[0]:
            raise IndexError("a sequence's block-table row is outside the table")

    def forward_layer_tree(self, plan: TreePlan, layer: int, x: torch.Tensor, out: torch.Tensor,
                           weights: "DeviceLayerWeights", mask: Optional[torch.Tensor],
                           block_tables: torch.Tensor,
                           rope_positions: Optional[torch.Tensor] = None, eps: float = 1e-5,
                           freq_base: float = 10000.0, neox: bool = False,
                           scale: Optional[float] = None, stream=None):
        """One transformer layer for the plan's drafted tokens (kvc_forward_layer_tree):
        x / out (tokens, hidden) fp16; rope_positions (tokens) int32, context + depth of
        each token (None: its cache slot, right for a chain).  out may be x."""
        dev, t = self.device, plan.n_tokens
        n = t * weights.hidden
        sc = default_scale(self.head_dim) if scale is None else float(scale)
        if len(weights.w) != 7 or len(weights.types) != 7:
            raise ValueError("a layer has seven weights: q, k, v, o, gate, up, down")
        for w in weights.w:
            if w.get_device() != dev or not w.is_contiguous():
                raise ValueError(f"weights must be contiguous tensors on cuda:{dev}")
        wt = [x for w, ty in zip(weights.w, weights.types) for x in (int(w.data_ptr()), int(ty))]
        mp, words = self._mask(mask, t)
        self._table(block_tables, plan)
        ffi.check(ffi.lib.kvc_forward_layer_tree(
            self.handle, plan.handle, layer, _on(x, "x", torch.float16, n, dev),
            _on(out, "out", torch.float16, n, dev),
            _on(weights.attn_norm, "attn_norm", torch.float16, weights.hidden, dev), *wt[:8],
            _on(weights.ffn_norm, "ffn_norm", torch.float16, weights.hidden, dev), *wt[8:], mp,
            words,
            None if rope_positions is None else _on(rope_positions, "rope_positions", torch.int32,
                                                    t, dev),
            block_tables.data_ptr(), block_tables.shape[0], block_tables.shape[1], weights.hidden,
            weights.intermediate, float(eps), float(freq_base), 1 if neox else 0, sc,
            _stream_on(stream, dev)))

    def commit_tree(self, block_tables: torch.Tensor, ctx_lens: torch.Tensor,
                    paths: torch.Tensor, path_lens: torch.Tensor,
                    rows: Optional[torch.Tensor] = None, stream=None):
        """Move the accepted paths' rows together in every layer (kvc_commit_tree):
        the row of slot ctx_lens[i] + paths[i, j] goes to slot ctx_lens[i] + j.  All int32
        CUDA tensors; paths (sequences, longest), ascending; rows default to i."""
        dev, n = self.device, path_lens.numel()
        if paths.dim() != 2 or block_tables.dim() != 2:
            raise ValueError("paths and block_tables must have two dimensions")
        if paths.shape[0] != n:
            raise ValueError("paths needs one row per sequence")
        if rows is None and n > block_tables.shape[0]:
            raise IndexError("a sequence's block-table row is outside the table")
        ffi.check(ffi.lib.kvc_commit_tree(
            self.handle, _on(block_tables, "block_tables", torch.int32, 0, dev),
            block_tables.shape[0], block_tables.shape[1],
            None if rows is None else _on(rows, "rows", torch.int32, n, dev),
            _on(ctx_lens, "ctx_lens", torch.int32, n, dev),
            _on(paths, "paths", torch.int32, 0, dev), paths.shape[1],
            _on(path_lens, "path_lens", torch.int32, 0, dev), n, _stream_on(stream, dev)))

    def reorder_beams(self, block_tables: torch.Tensor, parents: torch.Tensor,
                      ctx_lens: torch.Tensor, stream=None):
        """Let the beams' cached states follow their parents, in place
        (kvc_reorder_beams): block_tables (sequences * beams, pages), parents
        (sequences, beams) and ctx_lens (sequences), int32 CUDA tensors."""
        dev = self.device
        if parents.dim() != 2 or block_tables.dim() != 2:
            raise ValueError("parents and block_tables must have two dimensions")
        n, beams = parents.shape
        if block_tables.shape[0] != n * beams:
            raise ValueError("block_tables needs one row per beam")
        ffi.check(ffi.lib.kvc_reorder_beams(
            self.handle, _on(block_tables, "block_tables", torch.int32, 0, dev),
            block_tables.shape[1], _on(parents, "parents", torch.int32, 0, dev),
            _on(ctx_lens, "ctx_lens", torch.int32, n, dev), n, beams, _stream_on(stream, dev)))

    def gather(self, layer: int, block_tables: torch.Tensor, row: int, start: int, count: int,
               stream=None):
        with _made_on(stream, self.device):
            k = torch.empty((count, self.num_kv_heads, self.head_dim), dtype=self.dtype,
                            device=f"cuda:{self.device}")
            v = torch.empty_like(k)
        ffi.check(ffi.lib.kvc_gather(self.handle, layer, _i32(block_tables),
                                     int(block_tables.shape[-1]), row, start, count,
                                     int(k.data_ptr()), int(v.data_ptr()), _sp(stream)))
        return k, v

    def close(self):
        if self.handle is not None:
            ffi.check(ffi.lib.kvc_pool_destroy(self.handle))
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


@dataclass
class DeviceLayerWeights:
    """One transformer layer's weights resident on the GPU: the two RMSNorm
    weights ((hidden,) fp16) and the seven GGML-typed weights (raw block bytes,
    kvc_weight_bytes long) in the order q, k, v, o, gate, up, down, with their
    type ids (KVC_WTYPE_*), as forward_layer_cached takes them."""
    attn_norm: torch.Tensor
    ffn_norm: torch.Tensor
    w: Sequence[torch.Tensor]
    types: Sequence[int]
    hidden: int
    intermediate: int


class BatchDecoder:
    """The decode loop of generate_batch_ids (src/inference.py:435-447) on the
    paged pool: the reference decodes its prompts one after another, one
    forward_layer_cached call per (sequence, layer, token); here every sequence
    of the batch advances by one token per step, one kvc_forward_layer_paged
    call per layer for the whole batch.  Sequence i owns block-table row i;
    ``ctx_lens[i]`` counts its cached positions.  The embedding lookup, the
    final norm, the LM head and sampling stay with the caller.

    With ``stream`` a call's whole work runs there: its inputs must be ready on that
    stream, and what it returns belongs to it, as after ``torch.cuda.stream(stream)``."""

    def __init__(self, cache: PagedKVCache, layers: Sequence[DeviceLayerWeights],
                 block_tables: torch.Tensor, num_heads: int, ctx_lens: Sequence[int],
                 eps: float = 1e-5, freq_base: float = 10000.0, neox: bool = False,
                 scale: Optional[float] = None):
        if len(layers) != cache.num_layers:
            raise ValueError("one DeviceLayerWeights per pool layer is required")
        if block_tables.dim() != 2 or block_tables.shape[0] < len(ctx_lens):
            raise ValueError("block_tables needs one row per sequence")
        self.cache, self.layers, self.bt = cache, list(layers), block_tables
        self.num_heads = int(num_heads)
        self.ctx = np.asarray(ctx_lens, dtype=np.int64).copy()
        self.eps, self.freq_base, self.neox, self.scale = eps, freq_base, neox, scale
        self.plan = DecodePlan()
        self.tree_plan: Optional[TreePlan] = None
        self._drafted: Optional[list] = None      # node counts of the last verify
        self.capacity = int(block_tables.shape[1]) * cache.page_size

    def prefill(self, seq: int, x: torch.Tensor, stream=None) -> torch.Tensor:
        """Run tokens x (n, hidden) of sequence `seq` at positions ctx_lens[seq]..
        through every layer (causal over the cached prefix and the chunk itself);
        returns the last layer's output (n, hidden)."""
        n = int(x.shape[0])
        if n == 0:
            return x
        p0 = int(self.ctx[seq])
        if p0 + n > self.capacity:
            raise IndexError("prefill exceeds the sequence's block-table capacity")
        self.cache.plan(np.arange(p0 + 1, p0 + n + 1), self.num_heads, rows=[seq] * n,
                        plan=self.plan, stream=stream)
        y = self._layers(x, stream)
        self.ctx[seq] += n
        return y

    def step(self, x: torch.Tensor, stream=None) -> torch.Tensor:
        """One decode step: token i of x (batch, hidden) is sequence i's next token
        at position ctx_lens[i]; returns the last layer's output (batch, hidden)."""
        b = len(self.ctx)
        if int(x.shape[0]) != b:
            raise ValueError(f"x must hold one token per sequence ({b})")
        if int(self.ctx.max(initial=0)) + 1 > self.capacity:
            raise IndexError("a sequence would exceed its block-table capacity")
        self.cache.plan(self.ctx + 1, self.num_heads, plan=self.plan, stream=stream)
        y = self._layers(x, stream)
        self.ctx += 1
        return y

    def verify(self, x: torch.Tensor, trees: Sequence[Sequence[int]], stream=None) -> torch.Tensor:
        """Run drafted tokens through every layer: trees[i] holds the parents of sequence
        i's drafted tokens (tree_masks; empty for none), x (tokens, hidden) their
        embeddings, sequence by sequence.  Each token attends over its sequence's
        cached context, its ancestors and itself; returns the last layer's output
        (tokens, hidden).  The context lengths stay until ``commit`` keeps a path."""
        b = len(self.ctx)
        if len(trees) != b:
            raise ValueError(f"one tree per sequence is required ({b})")
        counts = [len(t) for t in trees]
        n = sum(counts)
        if int(x.shape[0]) != n:
            raise ValueError(f"x must hold one row per drafted token ({n})")
        for c, k in zip(self.ctx, counts):
            if k and int(c) + k > self.capacity:
                raise IndexError("a tree exceeds its sequence's block-table capacity")
        words = max(1, (max(counts, default=0) + 31) // 32)
        masks = [tree_masks(t, words) for t in trees]
        self._drafted = None
        if n == 0:
            self._drafted = counts
            return x
        pos = np.concatenate([int(c) + tree_depths(t) for c, t in zip(self.ctx, trees)])
        with _made_on(stream, self.bt.device):
            mask = _upload(np.concatenate(masks), x.device)
            rope_pos = _upload(pos.astype(np.int32), x.device)
            cur = x.contiguous()
            bufs = (torch.empty_like(cur), torch.empty_like(cur))   # x itself is never written
        self.tree_plan = self.cache.plan_tree(self.ctx, counts, self.num_heads,
                                              plan=self.tree_plan, stream=stream)
        for layer, lw in enumerate(self.layers):
            nxt = bufs[layer % 2]
            self.cache.forward_layer_tree(self.tree_plan, layer, cur, nxt, lw, mask, self.bt,
                                          rope_pos, self.eps, self.freq_base, self.neox,
                                          self.scale, stream)
            cur = nxt
        self._drafted = counts
        return cur

    def commit(self, paths: Sequence[Sequence[int]], stream=None) -> None:
        """Keep paths[i], ascending node numbers of sequence i's last ``verify`` (empty:
        none): their rows move together behind the context, which grows by them."""
        if self._drafted is None:
            raise RuntimeError("commit needs the trees of a verify before it")
        if len(paths) != len(self.ctx):
            raise ValueError(f"one path per sequence is required ({len(self.ctx)})")
        for p, k in zip(paths, self._drafted):
            if any(not 0 <= a < k for a in p) or any(a >= b for a, b in zip(p, p[1:])):
                raise ValueError("a path holds ascending numbers of its tree's nodes")
        lens = np.array([len(p) for p in paths], dtype=np.int32)
        if lens.max(initial=0) > 0:
            mat = np.zeros((len(paths), int(lens.max())), dtype=np.int32)
            for i, p in enumerate(paths):
                mat[i, :len(p)] = p
            with _made_on(stream, self.bt.device):
                ctx, mat, n = (_upload(a, self.bt.device)
                               for a in (self.ctx.astype(np.int32), mat, lens))
            self.cache.commit_tree(self.bt, ctx, mat, n, stream=stream)
        self.ctx += lens
        self._drafted = None

    def reorder(self, parents: np.ndarray, stream=None) -> None:
        """Beam search: rows are sequences * beams, parents (sequences, beams) beam
        numbers; every row takes its parent's cached states (reorder_beams).  The
        block table is permuted in place: give the decoder one of its own.  The rows of
        a ``verify`` that was not committed do not follow: it is dropped."""
        parents = np.ascontiguousarray(np.asarray(parents, dtype=np.int32))
        if parents.ndim != 2 or parents.size != len(self.ctx):
            raise ValueError("parents needs one entry per row, (sequences, beams)")
        n, beams = parents.shape
        if parents.size and (parents.min() < 0 or parents.max() >= beams):
            raise ValueError("a parent is not a beam of its sequence")
        ctx = self.ctx.reshape(n, beams)
        if np.any(ctx != ctx[:, :1]):
            raise ValueError("the beams of a sequence must have the same context length")
        with _made_on(stream, self.bt.device):
            par = _upload(parents, self.bt.device)
            lens = _upload(ctx[:, 0].astype(np.int32), self.bt.device)
        self._drafted = None      # (drafted rows lie behind the positions that move)
        # (the table may have rows behind the decoder's)
        self.cache.reorder_beams(self.bt[:parents.size], par, lens, stream=stream)

    def _layers(self, x: torch.Tensor, stream) -> torch.Tensor:
        with _made_on(stream, self.bt.device):
            cur = x.contiguous()
            bufs = (torch.empty_like(cur), torch.empty_like(cur))   # x itself is never written
        for layer, lw in enumerate(self.layers):
            nxt = bufs[layer % 2]
            self.cache.forward_layer(self.plan, layer, cur, nxt, lw, self.bt, self.eps,
                                     self.freq_base, self.neox, self.scale, stream)
            cur = nxt
        self._drafted = None
        return cur

    def close(self):
        self.plan.close()
        if self.tree_plan is not None:
            self.tree_plan.close()


# -- drafted trees --------------------------------------------------------------------
def tree_masks(parents: Sequence[int], words: Optional[int] = None) -> np.ndarray:
    """Mask rows (nodes, words) int32 of one drafted tree for decode_tree: node i sees
    itself and its ancestors.  parents[i] is the node above i, smaller than i, or -1."""
    n = len(parents)
    need = max(1, (n + 31) // 32)
    words = need if words is None else int(words)
    if n > ffi.MAX_TREE_NODES or words < need:
        raise ValueError(f"{n} nodes do not fit {words} mask words or the limit of "
                         f"{ffi.MAX_TREE_NODES}")
    m = np.zeros((n, words), dtype=np.uint32)
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError("a node's parent must be drafted before it (or be -1)")
        if p >= 0:
            m[i] = m[p]
        m[i, i // 32] |= np.uint32(1 << (i % 32))
    return m.view(np.int32)


def tree_depths(parents: Sequence[int]) -> np.ndarray:
    """Depth of each node: 0 for a node right behind the context."""
    d = np.zeros(len(parents), dtype=np.int32)
    for i, p in enumerate(parents):
        d[i] = 0 if p < 0 else d[p] + 1
    return d


# -- layout helpers -------------------------------------------------------------------
def rope(x: torch.Tensor, out: torch.Tensor, positions: Optional[torch.Tensor] = None,
         pos_offset: int = 0, freq_base: float = 10000.0, neox: bool = False, stream=None):
    """Rotary position embedding of x (tokens, heads, D) into out on the GPU
    (kvc_rope); token t at positions[t] (int32 CUDA tensor) or pos_offset + t."""
    if x.dim() != 3:
        raise ValueError("x must be (tokens, heads, head_dim)")
    n, heads, d = x.shape
    dt = _TORCH_CODE.get(x.dtype)
    if dt is None:
        raise ValueError(f"unsupported dtype {x.dtype}")
    xp = _dev(x, "x", x.dtype, n * heads * d)
    op = _dev(out, "out", x.dtype, n * heads * d)
    pp = None if positions is None else _i32(positions)
    ffi.check(ffi.lib.kvc_rope(xp, op, n, heads, d, pp, int(pos_offset), float(freq_base),
                               int(bool(neox)), dt, _sp(stream)))
    return out


def pages_for(ctx_lens: Sequence[int], page_size: int) -> np.ndarray:
    return np.array([(int(c) + page_size - 1) // page_size for c in ctx_lens], dtype=np.int64)


def random_block_tables(ctx_lens: Sequence[int], page_size: int, seed: int):
    """Block tables for sequences of the given lengths over a pool with exactly
    the pages they need, assigned in a seeded random permutation (benchmark
    config 3: "paged fp16 pool of 16-token pages with a random page permutation").
    Returns (table (n, max_pages) int32 numpy, total pages)."""
    need = pages_for(ctx_lens, page_size)
    total = int(need.sum())
    perm = np.random.default_rng(seed).permutation(total).astype(np.int32)
    width = int(need.max()) if len(need) else 1
    table = np.full((len(need), max(1, width)), -1, dtype=np.int32)
    o = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[o:o + n]
        o += int(n)
    # unused tail entries point at page 0 (never read: beyond every context)
    table[table < 0] = 0
    return table, total


def shard_heads(num_kv_heads: int, world: int, rank: int):
    """KV heads [h0, h1) owned by `rank` when heads are split across `world` GPUs."""
    from sharding import shard_heads as _shard

    return _shard(num_kv_heads, world, rank)


def default_scale(head_dim: int) -> float:
    """1/sqrt(head_dim), the scale every caller passes (src/layer.py:181)."""
    return 1.0 / math.sqrt(head_dim)
