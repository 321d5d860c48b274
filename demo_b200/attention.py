"""Attention over a paged KV cache (include/kvattn.h) for torch tensors:
single tokens, chains and trees of drafted tokens, straight from the pages that
the cache manager loads and stores.

CrossCache leaves attention to the engine; the paged geometries are those of
cache.layout_from_kv_tensors (vLLM's FlashAttention and FlashInfer layouts).
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Sequence

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _lib
from ._lib import KvAttnDesc, lib
from .cache import CacheError, KVLayout
from .pages import _current_stream, _int32, _on_stream, _used_on, planes_on

# struct kv_attn_desc in one go: 12 pointers, 8 64-bit numbers, 12 32-bit ones, three floats, the device
_DESC = struct.Struct("@12PQQqqqqq10I2i3fi")
_TYPES = {torch.bfloat16: _lib.KVATTN_BF16, torch.float16: _lib.KVATTN_FP16}
_KV_TYPES = {**_TYPES, torch.float8_e4m3fn: _lib.KVATTN_E4M3}
_BYTES = (torch.uint8, torch.int8, torch.int16, torch.uint16)      # tensors that say nothing about their values

_ERRORS = ((_lib.KVATTN_ERR_PAGE, "a page id outside the cache"),
           (_lib.KVATTN_ERR_SEQ, "offsets out of order, or a row or length that fits neither table nor nodes"),
           (_lib.KVATTN_ERR_PARENT, "a parent that does not come before its node"),
           (_lib.KVATTN_ERR_TIMEOUT, "a wait inside the kernel ran out"))


class TreeAttention:
    """Attention of fed tokens over the layers of one paged cache.

    layout, k_ptrs, v_ptrs: from cache.layout_from_kv_tensors; K and V planes
        of 16-bit values of the queries' type, or of float8_e4m3fn values that
        k_scale and v_scale bring back
    kv_dtype: the values' type where the layout's tensors do not say it (8-bit
        caches that an engine keeps as uint8).  A layout made by hand, without
        a dtype, stands for float8_e4m3fn or the queries' type, by its element size
    num_heads, num_kv_heads: query heads and K/V heads of this rank
    scale: of the scores, by default head_dim ** -0.5
    """

    def __init__(self, layout: KVLayout, k_ptrs: Sequence[int], v_ptrs: Sequence[int], num_heads: int, num_kv_heads: int,
                 scale: float | None = None, k_scale: float = 1.0, v_scale: float = 1.0, kv_dtype: torch.dtype | None = None):
        if layout.kv != 2 or v_ptrs is None:
            raise ValueError("attention needs K and V planes (a K-only latent cache is not supported)")
        if len(k_ptrs) != layout.num_layers or len(v_ptrs) != layout.num_layers:
            raise ValueError("one pointer per layer")
        if num_kv_heads < 1 or num_heads % num_kv_heads or layout.hidden_dim_size % num_kv_heads:
            raise ValueError("num_kv_heads must divide num_heads and the layout's width")
        if layout.element_size not in (1, 2):
            raise ValueError("caches of 1 or 2-byte elements")
        held = layout.dtype
        if kv_dtype is not None:
            if held is not None and held is not kv_dtype and held not in _BYTES:
                raise ValueError(f"kv_dtype: the cache holds {held}, not {kv_dtype}")
            held = kv_dtype
        elif held is None and layout.element_size == 1:
            held = torch.float8_e4m3fn
        if held is not None and (held not in _KV_TYPES or held.itemsize != layout.element_size):
            raise ValueError(f"caches of bfloat16, float16 or float8_e4m3fn values, not {held}"
                             + (" (kv_dtype says what bytes stand for)" if held in _BYTES else ""))
        if num_heads // num_kv_heads > 128:
            raise ValueError("at most 128 query heads per K/V head")
        dim = layout.hidden_dim_size // num_kv_heads
        if layout.head_bytes and layout.head_bytes != dim * layout.element_size:
            raise ValueError("num_kv_heads does not fit the layout's head-major pages")
        if dim % 16 or dim > _lib.KVATTN_MAX_HEAD_DIM:
            raise ValueError(f"head_dim must be a multiple of 16 up to {_lib.KVATTN_MAX_HEAD_DIM} (got {dim})")
        if any(not p or p % 16 for p in (*k_ptrs, *v_ptrs)) or layout.block_stride % 16:
            raise ValueError("planes and pages must be 16-byte aligned")
        scale = dim ** -0.5 if scale is None else float(scale)
        if not (0 < scale * k_scale < math.inf) or not 0 < scale < math.inf or not math.isfinite(v_scale):
            raise ValueError("scale and k_scale must be finite and above 0, v_scale finite")
        self.layout, self.num_heads, self.num_kv_heads, self.head_dim = layout, num_heads, num_kv_heads, dim
        self._k, self._v = [int(p) for p in k_ptrs], [int(p) for p in v_ptrs]
        self._devices: dict[int, tuple[torch.Tensor, int, int]] = {}     # error bits, their address, workspace bytes
        self._shape = (layout.num_blocks, layout.block_size, num_heads, num_kv_heads, dim, 1 if layout.head_bytes else 0)
        self._scales = (scale, float(k_scale), float(v_scale))
        self.kv_dtype = held                # None: the queries'
        if torch.cuda.is_initialized() and not torch.cuda.is_current_stream_capturing():
            at = lib.kv_page_device_of(self._k[0])      # else its first call will say what is wrong with it
            if at >= 0 or at == _lib.KVPAGE_ANY_DEVICE:
                self._device(at if at >= 0 else torch.cuda.current_device())

    def _device(self, index: int) -> tuple[torch.Tensor, int, int]:
        planes_on(index, (*self._k, *self._v))
        d = KvAttnDesc(table_stride=1, width=1, num_rows=1, device=index, scale=self._scales[0], k_scale=self._scales[1])
        d.num_pages, d.block_size, d.num_heads, d.num_kv_heads, d.head_dim, d.head_major = self._shape
        need = lib.kv_attn_workspace_bytes(C.addressof(d))
        if need < 0:
            raise CacheError("kv_attn_workspace_bytes", need)
        with torch.cuda.device(index):
            if torch.cuda.is_current_stream_capturing():
                raise ValueError(f"the first call on cuda:{index} cannot be captured")
            error = torch.zeros(1, dtype=torch.int32, device="cuda")
            torch.cuda.current_stream().synchronize()   # the call may be on another stream
        self._devices[index] = found = error, error.data_ptr(), need
        return found

    def __call__(self, layer: int, q: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 q_offsets: torch.Tensor, parents: torch.Tensor | None = None, rows: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, return_lse: bool = False, stream: torch.cuda.Stream | None = None):
        """out [total, num_heads, head_dim] (and lse [total, num_heads] in
        float32) of the packed queries q, both as q's type and layout say.

        q            bfloat16 or float16 [total, num_heads, head_dim], CUDA
        block_table  int32 [rows, width]; seq_lens int32 [rows], the fed tokens included
        q_offsets    int32 [sequences + 1]: sequence b feeds q[q_offsets[b]:q_offsets[b + 1]]
        parents      int32 [total]: the tree (-1: the last token before the fed
                     ones, -2: padding); None: a chain
        rows         int32 [sequences]: their rows; None: row b

        Runs on `stream`, by default the current stream of q's device, to which
        the results then belong.  With `stream` the arguments may be dropped when
        the call returns (on the current stream torch's own rules hold); the
        object must outlive its calls, and the graphs that captured them.  Queries that no sequence covers leave their rows of out and lse as
        they were, which in new tensors is anything.  May be
        captured, except for the first call of an object that was made before
        CUDA was used.
        """
        if (q.requires_grad and torch.is_grad_enabled()) or unpack_dual(q).tangent is not None:
            raise ValueError("q: attention over a cache has no gradients; call it under torch.no_grad(), without a tangent")
        if torch.jit.is_tracing():
            raise ValueError("attention over a cache cannot be traced: it would become a constant")
        index, kind = q.get_device(), _TYPES.get(q.dtype)
        if index < 0 or kind is None or q.dim() != 3 or q.shape[1] != self.num_heads or q.shape[2] != self.head_dim or \
                q.stride(2) != 1:
            raise ValueError(f"q: expected a bfloat16 or float16 CUDA tensor [total, {self.num_heads}, {self.head_dim}]")
        kv_type = kind if self.kv_dtype is None else _KV_TYPES[self.kv_dtype]
        if kv_type != kind and kv_type != _lib.KVATTN_E4M3:
            raise ValueError(f"q: {q.dtype} queries over a cache of {self.kv_dtype}")
        if stream is not None:
            caller = torch.cuda.current_stream(index)
            with _on_stream(stream, index):
                res = self(layer, q, block_table, seq_lens, q_offsets, parents, rows, out, return_lse)
            for t in res if return_lse else (res,):
                t.record_stream(caller)     # which may be where it is used and dropped
            _used_on(stream, q, block_table, seq_lens, q_offsets, parents, rows, out)
            return res
        total = q.shape[0]
        q_strides = q.stride()
        if 0 in q_strides:                              # an expanded tensor
            q = q.contiguous()
            q_strides = q.stride()
        if block_table.dim() != 2 or block_table.dtype is not torch.int32 or block_table.get_device() != index or \
                block_table.shape[1] < 1 or block_table.stride(1) != 1:
            raise ValueError(f"block_table: expected an int32 tensor [rows, width] on cuda:{index} with contiguous rows")
        n_rows, width = block_table.shape
        seqs = q_offsets.numel() - 1
        if seqs < 0 or (rows is None and seqs > n_rows):
            raise ValueError("q_offsets: expected one offset per sequence and the end")
        if out is None:
            out = torch.empty((total, self.num_heads, self.head_dim), dtype=q.dtype, device=q.device)
        elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != index or out.stride(2) != 1:
            raise ValueError("out: expected a tensor like q")
        out_strides = out.stride()
        lse = torch.empty((total, self.num_heads), dtype=torch.float32, device=q.device) if return_lse else None
        _, error, need = self._devices.get(index) or self._device(index)
        work = torch.empty(need, dtype=torch.uint8, device=q.device)    # of this call alone, also where graphs are captured
        row = self.num_heads * self.head_dim            # a stride of one row or one head means nothing
        pages, block, heads, kv_heads, dim, head_major = self._shape
        desc = _DESC.pack(
            q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, self._k[layer], self._v[layer],
            block_table.data_ptr(), _int32("seq_lens", seq_lens, index, n_rows),
            _int32("rows", rows, index, seqs) if rows is not None else 0, _int32("q_offsets", q_offsets, index),
            _int32("parents", parents, index, total) if parents is not None else 0, error, work.data_ptr(),
            need, self.layout.block_stride, block_table.stride(0) if n_rows > 1 else width,
            q_strides[0] if total > 1 else row, q_strides[1] if heads > 1 else row,
            out_strides[0] if total > 1 else row, out_strides[1] if heads > 1 else row,
            width, n_rows, seqs, total, pages, block, heads, kv_heads, dim, head_major, kind,
            kv_type, *self._scales, index)
        ret = lib.kv_attn_launch(desc, _current_stream(index))
        if ret:
            raise CacheError("kv_attn_launch", ret)
        return (out, lse) if return_lse else out

    def check(self) -> None:
        """Wait for the device and raise ValueError for what the calls since
        the last check() found wrong in their arguments."""
        for index, (error, _, _) in self._devices.items():
            torch.cuda.synchronize(index)       # calls on all streams
            bits = int(error.item())
            if bits:
                error.zero_()
                torch.cuda.synchronize(index)
                raise ValueError("tree attention: " + "; ".join(text for bit, text in _ERRORS if bits & bit))


__all__ = ["TreeAttention"]
