"""Paged attention of rows that see something else than a causal window: sliding windows whose first tokens stay
visible, and trees of drafted tokens.  ``paged_attention(sink_tokens=..., tree_mask=...)`` comes here.

A row's *visible sequence* is the context followed by the new tokens its mask names, in slot order (a causal row: those
up to itself).  A sliding window keeps its last ``sliding_window`` entries and ``sink_tokens`` its first ones; a row
that sees nothing gets zeros.
"""

from __future__ import annotations

import math
import typing as tp

import torch

from ... import _native as nv
from .unified_attention import (_CHECK, _TILED_BLOCK_SIZE_AFFINE, _TILED_BLOCK_SIZES_FLOAT, _TILED_HEAD_DIMS, _as_int32,
                                _make_pool, _scratch, _validate_inputs)


_status: dict = {}


def _status_word(device) -> torch.Tensor:
    """One word per device that every call ORs its faults into (a captured call must not bring a fill of its own)."""
    word = _status.get(device)
    if word is None:
        word = _status[device] = torch.zeros(1, dtype=torch.int32, device=device)
    return word


class VisibleAttentionCall:
    """One validated call, split like ``AttentionCall`` into ``plan()`` (work list) and ``launch()``.

    Work list and workspace belong to the call (the counters in them are set up by the work list), so calls on different
    streams and captured graphs share nothing but the status word."""

    def __init__(self, queries, key_cache, value_cache, block_tables, kv_lens, query_start_loc, *,
                 softmax_scale: float | None = None, sliding_window: int | None = None, sink_tokens: int = 0, tree_mask=None,
                 tree_seqs=None, k_scale=None, v_scale=None, k_bias=None, v_bias=None, kernel: str | None = None,
                 max_query_len: int = 0, plan=None, query_len_set: tp.Sequence[int] | None = None, long_seqs: int = 0):
        from ...caching.paged.cache import VisiblePlan, absent_row_classes, native_visibility, tree_arguments, visible_plan_flags

        nv.require_cuda(queries, key_cache, value_cache)
        dev = queries.device
        if key_cache.device != dev or value_cache.device != dev:
            raise ValueError("queries, key_cache and value_cache must be on one device")
        affine = key_cache.dtype == torch.uint8
        self.block_tables, self.kv_lens = _as_int32(block_tables, dev), _as_int32(kv_lens, dev)
        self.query_start_loc = _as_int32(query_start_loc, dev)
        _validate_inputs(queries, key_cache, value_cache, self.block_tables, self.kv_lens, self.query_start_loc, affine)
        if not (key_cache.is_contiguous() and value_cache.is_contiguous()):
            raise ValueError("key_cache and value_cache must be contiguous")
        if kernel not in (None, "generic", "tiled"):
            raise ValueError("a call with sinks or a tree takes kernel=None, 'generic' or 'tiled'")
        if int(sink_tokens) < 0 or int(sliding_window or 0) < 0:
            raise ValueError("sink_tokens and sliding_window must be non-negative")
        self.device = dev
        self.total, self.hq, self.d = (int(x) for x in queries.shape)
        self.num_seqs = int(self.block_tables.shape[0])
        if self.kv_lens.shape[0] != self.num_seqs:
            raise ValueError("kv_lens must have length num_seqs")
        self.tree_mask, self.tree_seqs = tree_arguments(tree_mask, tree_seqs, self.total, self.num_seqs, dev)
        if self.tree_mask is not None and tree_seqs is None and query_len_set:
            longest = max(int(x) for x in query_len_set)
            if longest > 64 * self.tree_mask.shape[1]:
                raise ValueError(f"a tree of {longest} tokens needs {-(-longest // 64)} mask words, got {self.tree_mask.shape[1]}")
        self.window, self.sinks = int(sliding_window or 0), int(sink_tokens)
        self.queries = queries.contiguous()
        if self.queries.data_ptr() % 16:
            self.queries = self.queries.clone()  # a view into the middle of a row: the tensor core's copies start on 16 bytes
        self.out: torch.Tensor | None = None
        if self.total == 0:
            return
        self.key_cache, self.value_cache = key_cache, value_cache
        self.scales = (k_scale, v_scale, k_bias, v_bias)
        self.pool, _ = _make_pool(key_cache, value_cache, self.d, k_scale, v_scale, k_bias, v_bias)
        tiled_ok = (
            (self.pool.block_size == _TILED_BLOCK_SIZE_AFFINE if affine else self.pool.block_size in _TILED_BLOCK_SIZES_FLOAT)
            and self.d in _TILED_HEAD_DIMS
            and queries.dtype in (torch.float16, torch.bfloat16)
            and (affine or key_cache.dtype == queries.dtype)
            and (key_cache.data_ptr() | value_cache.data_ptr()) % 16 == 0
        )
        if kernel == "tiled" and not tiled_ok:
            raise NotImplementedError(
                "the tiled kernels need page size 128 (or 16/32/64 with a 16-bit pool), head_dim 64 or 128, fp16/bf16 queries and a pool of "
                "the same dtype (or an affine pool)")
        self.kernel = kernel or ("tiled" if tiled_ok else "generic")
        self.visibility = native_visibility(self.sinks, self.tree_mask, self.tree_seqs)
        self.status = _status_word(dev)
        a = nv.AttnArgs()
        a.queries = self.queries.data_ptr()
        a.block_tables, a.kv_lens = self.block_tables.data_ptr(), self.kv_lens.data_ptr()
        a.query_start_loc = self.query_start_loc.data_ptr()
        a.total_tokens, a.num_seqs, a.num_q_heads = self.total, self.num_seqs, self.hq
        a.max_blocks_per_seq, a.q_dtype = int(self.block_tables.shape[1]), nv.dtype_code(queries.dtype)
        a.sliding_window = self.window
        a.softmax_scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(self.d)
        a.max_query_len = max(0, int(max_query_len))
        a.status = self.status.data_ptr()
        self.args = a
        if self.kernel == "generic":
            return
        lib, hkv = nv.lib(), self.pool.num_kv_heads
        words = 0 if self.tree_mask is None else int(self.tree_mask.shape[1])
        flags = visible_plan_flags(self.pool.kv_format, self.hq, hkv, self.d, int(long_seqs))
        self.plan_bytes = int(lib.emlx_visible_plan_bytes(self.num_seqs, self.total, self.hq, hkv, words))
        if query_len_set:
            flags |= absent_row_classes(query_len_set, self.hq // hkv, bool(flags & 1))
        self.planned = (isinstance(plan, VisiblePlan) and plan.num_q_heads == self.hq and plan.sliding_window == self.window
                        and plan.sink_tokens == self.sinks and plan.flags == flags and plan.buffer.numel() >= self.plan_bytes
                        and plan.tree_mask is self.tree_mask and plan.tree_seqs is self.tree_seqs)
        self.plan_buf = plan.buffer if self.planned else torch.empty(self.plan_bytes, dtype=torch.uint8, device=dev)
        a.plan_flags = flags
        a.row_class_mask = ~(flags >> 16) & 15 if flags >> 16 else 0
        ws_bytes = int(lib.emlx_visible_workspace_bytes(self.hq, hkv, self.d, int(a.max_query_len), flags))
        if affine and flags & 1:
            ws_bytes += int(lib.emlx_attn_dequant_bytes(self.pool, self.num_seqs, int(self.block_tables.shape[1]), int(long_seqs),
                                                        self.total, self.hq, nv.dtype_code(queries.dtype)))
        self.workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        a.plan, a.plan_bytes = self.plan_buf.data_ptr(), self.plan_bytes
        a.workspace, a.workspace_bytes = self.workspace.data_ptr(), ws_bytes

    def plan(self) -> "VisibleAttentionCall":
        if self.total and self.kernel != "generic" and not self.planned:
            with nv.on_device(self.device):
                nv.check(nv.lib().emlx_visible_plan(
                    nv.ptr(self.query_start_loc), nv.ptr(self.kv_lens), self.num_seqs, self.total, self.hq,
                    self.pool.num_kv_heads, self.pool.block_size, self.window, self.visibility, int(self.args.max_query_len),
                    int(self.args.plan_flags), nv.ptr(self.plan_buf), self.plan_bytes, nv.ptr(self.status),
                    nv.stream_ptr(self.device)))
            self.planned = True
        return self

    def launch(self) -> torch.Tensor:
        if self.total == 0:
            return torch.zeros_like(self.queries)
        lib = nv.lib()
        self.out = torch.empty_like(self.queries)
        if _CHECK:
            self.out.fill_(float("nan"))  # a row no kernel writes shows up in the caller's checks
        self.args.out = self.out.data_ptr()
        with nv.on_device(self.device):
            entry = lib.emlx_attn_visible_generic if self.kernel == "generic" else lib.emlx_attn_visible
            nv.check(entry(self.args, self.pool, self.visibility, nv.stream_ptr(self.device)))
            if _CHECK and not torch.cuda.is_current_stream_capturing():
                rc = lib.emlx_read_status(nv.ptr(self.status), nv.stream_ptr(self.device))
                if rc != nv.EMLX_OK:
                    self.status.zero_()  # report once
                nv.check(rc)
        return self.out


__all__ = ("VisibleAttentionCall",)
