"""Device-resident pages of a paged KV cache (include/kvpage.h) for torch
block tables.

A PagePool owns the bookkeeping of an engine's paged cache: which row (a
sequence) holds which pages, how many rows share a page, which pages are free.
resize() allocates and frees, fork() shares a prefix, copy() moves pages,
compact() drops tokens out of rows (the rejected ones of a speculative step,
or evicted ones).  All of it stays on the GPU: no call reads anything back,
so an engine's step can be captured into a graph.  CrossCache leaves this to
the engine (its block ids come from vLLM, src/cache/cache.c:345-398).
"""
from __future__ import annotations

import ctypes as C
from typing import Sequence

import torch

from . import _lib
from ._lib import KvPageCache, KvPageState, lib
from .cache import CacheError, KVLayout

_ERRORS = ((_lib.KVPAGE_ERR_PAGE, "a page id outside the cache"),
           (_lib.KVPAGE_ERR_ROW, "a row outside the table, named twice, or of a length or state that the call cannot take"),
           (_lib.KVPAGE_ERR_REFS, "a page given back too often, or tokens moved into a shared page"),
           (_lib.KVPAGE_ERR_KEEP, "kept tokens not strictly ascending inside their row"),
           (_lib.KVPAGE_ERR_ALIGN, "a null or misaligned layer base"))

OK, NO_PAGES, INVALID = _lib.KVPAGE_OK, _lib.KVPAGE_NO_PAGES, _lib.KVPAGE_INVALID


# The calls are short on the GPU too: the helpers ask a tensor for its device's
# number and torch for the stream's handle, which costs a tenth of the objects.
_current_stream = torch._C._cuda_getCurrentRawStream


def _on_stream(stream: torch.cuda.Stream, index: int):
    """Context in which `stream` is the current one: what a call on it allocates
    is then ordered with it, where memory of another stream might still be in
    use there."""
    if stream.device_index != index:
        raise ValueError(f"stream: expected a stream of cuda:{index}")
    return torch.cuda.stream(stream)


def _used_on(stream: torch.cuda.Stream | None, *tensors: torch.Tensor | None) -> None:
    """What a call on `stream` was given: the caller may drop it when the call
    returns, and its memory must not be handed out again before the stream has
    come that far."""
    if stream is not None:
        for t in tensors:
            if t is not None:
                t.record_stream(stream)


def _int32(name: str, t: torch.Tensor, index: int, numel: int | None = None) -> int:
    """data pointer of a contiguous int32 tensor on CUDA device `index` (-1:
    the CPU); ValueError otherwise"""
    if t.dtype is not torch.int32 or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous int32 tensor on {f'cuda:{index}' if index >= 0 else 'the CPU'}")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name}: expected {numel} values, got {t.numel()}")
    return t.data_ptr()


def plane_bases(layout: KVLayout, k_ptrs: Sequence[int], v_ptrs: Sequence[int] | None,
                device: torch.device) -> tuple[torch.Tensor, torch.Tensor | None, int]:
    """Device arrays of the layers' K and V plane bases, and a power of two
    (at most 16) that divides every one of them."""
    if len(k_ptrs) != layout.num_layers or (v_ptrs is not None and len(v_ptrs) != layout.num_layers):
        raise ValueError("one pointer per layer")
    if (v_ptrs is None) != (layout.kv == 1):
        raise ValueError("layout.kv must be 1 exactly when v_ptrs is None")
    every = 16
    for p in (*k_ptrs, *(v_ptrs or ())):
        if not p:
            raise ValueError("a layer base is null")
        every |= int(p)
    both = torch.tensor([int(p) for p in (*k_ptrs, *(v_ptrs or ()))], dtype=torch.int64, device=device)
    return both[:layout.num_layers], both[layout.num_layers:] if v_ptrs is not None else None, every & -every


def planes_on(index: int, ptrs: Sequence[int]) -> None:
    """ValueError unless kernels on CUDA device `index` may follow every base"""
    for p in ptrs:
        at = lib.kv_page_device_of(p)
        if at < 0 and at != _lib.KVPAGE_ANY_DEVICE:
            raise ValueError("a layer base is not memory that a GPU reaches")
        if at not in (index, _lib.KVPAGE_ANY_DEVICE):
            raise ValueError(f"the cache is on cuda:{at}, not on cuda:{index}")


class PagePool:
    """The pages of one paged cache and the rows that hold them.

    layout, k_ptrs, v_ptrs: from cache.layout_from_kv_tensors (the planes
        themselves stay the caller's and must outlive the pool)
    block_table  int32 [rows, width], CUDA; rows may be strided
    seq_lens     int32 [rows]
    refs, free_list, free_count: the state to continue from (int32
        [num_blocks], [num_blocks], [1]); all three or none.  None starts with
        every page free, handed out from page 0 up, and needs empty rows.

    The tensors are updated in place and stay readable by the engine's own
    kernels.  Calls run on `stream`, by default the current stream of the
    cache's device, in the order they are made; calls for one pool on several
    streams have to be ordered by the caller, and results belong to the stream
    of their call.  The arguments of a call with `stream` may be dropped when it
    returns (on the current stream torch's own rules hold); the pool itself must
    outlive its calls, and the graphs that captured them.  The int32 results of
    resize, fork and compact say per row pages.OK, NO_PAGES or INVALID, on the
    device.
    """

    def __init__(self, layout: KVLayout, k_ptrs: Sequence[int], v_ptrs: Sequence[int] | None,
                 block_table: torch.Tensor, seq_lens: torch.Tensor, refs: torch.Tensor | None = None,
                 free_list: torch.Tensor | None = None, free_count: torch.Tensor | None = None):
        dev = block_table.device
        if dev.type != "cuda" or block_table.dtype is not torch.int32 or block_table.dim() != 2 or \
                block_table.shape[1] < 1 or block_table.shape[0] < 1 or block_table.stride(1) != 1 or \
                (block_table.shape[0] > 1 and block_table.stride(0) < block_table.shape[1]):
            raise ValueError("block_table: expected an int32 CUDA tensor [rows, width] with contiguous rows")
        rows, width = block_table.shape
        if rows > _lib.KVPAGE_MAX_ROWS:
            raise ValueError(f"at most {_lib.KVPAGE_MAX_ROWS} rows")
        if (refs is None) != (free_list is None) or (refs is None) != (free_count is None):
            raise ValueError("refs, free_list and free_count: all three or none")
        n = layout.num_blocks
        fresh = refs is None
        if fresh:
            refs = torch.zeros(n, dtype=torch.int32, device=dev)
            free_list = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=dev)
            free_count = torch.full((1,), n, dtype=torch.int32, device=dev)
        self.layout, self.device = layout, dev
        self.block_table, self.seq_lens = block_table, seq_lens
        self.refs, self.free_list, self.free_count = refs, free_list, free_count
        zeros = torch.zeros(1 + n, dtype=torch.int32, device=dev)
        self.error, self._marks = zeros[:1], zeros[1:]
        self._k, self._v, align = plane_bases(layout, k_ptrs, v_ptrs, dev)
        planes_on(dev.index, (*k_ptrs, *(v_ptrs or ())))
        self._index = index = dev.index
        lens = _int32("seq_lens", seq_lens, index, rows)
        if fresh and bool(seq_lens.any()):      # their pages would be handed out again
            raise ValueError("seq_lens: a pool that starts with every page free needs empty rows")
        self._state = KvPageState(
            table=block_table.data_ptr(), lens=lens,
            refs=_int32("refs", refs, index, n), free_list=_int32("free_list", free_list, index, n),
            free_count=_int32("free_count", free_count, index, 1), marks=self._marks.data_ptr(),
            error=self.error.data_ptr(), table_stride=block_table.stride(0) if rows > 1 else width, width=width,
            num_rows=rows, num_pages=n, block_size=layout.block_size, device=self._index)
        self._cache = KvPageCache(
            layer_k=self._k.data_ptr(), layer_v=self._v.data_ptr() if self._v is not None else None,
            error=self.error.data_ptr(), block_stride=layout.block_stride, unit_bytes=layout.unit,
            head_bytes=layout.head_bytes, block_size=layout.block_size, num_layers=layout.num_layers, num_pages=n,
            base_align=align, device=self._index)
        self._state_p, self._cache_p = C.addressof(self._state), C.addressof(self._cache)
        torch.cuda.current_stream(dev).synchronize()    # the first call may be on any stream

    def _results(self, n: int, scratch: int, stream) -> tuple[torch.Tensor, int]:
        """n results and `scratch` values behind them, and the stream's handle"""
        if stream is not None:
            caller = torch.cuda.current_stream(self.device)
            with _on_stream(stream, self._index):
                out, st = self._results(n, scratch, None)
            out.record_stream(caller)       # which may be where it is used and dropped
            return out, st
        return torch.empty(n + scratch, dtype=torch.int32, device=self.device), _current_stream(self._index)

    def resize(self, rows: torch.Tensor, lens: torch.Tensor, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Give row rows[i] the pages of lens[i] tokens (0 frees it): rows that
        shrink give pages back first, then rows that grow take theirs in the
        order of the call.  Returns each row's result."""
        n = rows.numel()
        status, st = self._results(n, 0, stream)
        ret = lib.kv_page_resize_launch(self._state_p, _int32("rows", rows, self._index),
                                        _int32("lens", lens, self._index, n), n, status.data_ptr(), st)
        if ret:
            raise CacheError("kv_page_resize_launch", ret)
        _used_on(stream, rows, lens)
        return status

    def copy(self, src: torch.Tensor, dst: torch.Tensor, tokens: torch.Tensor | None = None,
             stream: torch.cuda.Stream | None = None) -> None:
        """Copy page src[i] to page dst[i] in every layer (only its first
        tokens[i] tokens, with tokens).  Destinations are distinct and not
        among the sources."""
        n = src.numel()
        st = self._results(0, 0, stream)[1] if stream is not None else _current_stream(self._index)
        ret = lib.kv_page_copy_launch(self._cache_p, _int32("src", src, self._index), _int32("dst", dst, self._index, n),
                                      _int32("tokens", tokens, self._index, n) if tokens is not None else None, n, st)
        if ret:
            raise CacheError("kv_page_copy_launch", ret)
        _used_on(stream, src, dst, tokens)

    def fork(self, parents: torch.Tensor, children: torch.Tensor,
             stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Make each empty row children[i] a continuation of row parents[i]:
        full pages are shared, a partly filled last page is copied.  Returns
        each child's result."""
        n = parents.numel()
        out, st = self._results(n, 3 * n, stream)
        ret = lib.kv_page_fork_launch(self._cache_p, self._state_p, _int32("parents", parents, self._index),
                                      _int32("children", children, self._index, n), n, out.data_ptr() + 4 * n,
                                      out.data_ptr(), st)
        if ret:
            raise CacheError("kv_page_fork_launch", ret)
        _used_on(stream, parents, children)
        return out[:n]

    def compact(self, rows: torch.Tensor, start: torch.Tensor, keep: torch.Tensor, offsets: torch.Tensor,
                stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """In row rows[i] keep the tokens before start[i] and those at positions
        keep[offsets[i]:offsets[i + 1]] (ascending, from start[i] on), moved
        up behind them in every layer; the row's length follows and the pages
        left over are given back.  Returns each row's result."""
        n = rows.numel()
        out, st = self._results(n, n, stream)
        ret = lib.kv_page_compact_launch(self._cache_p, self._state_p, _int32("rows", rows, self._index),
                                         _int32("start", start, self._index, n), _int32("keep", keep, self._index),
                                         _int32("offsets", offsets, self._index, n + 1), keep.numel(), n,
                                         out.data_ptr() + 4 * n, out.data_ptr(), st)
        if ret:
            raise CacheError("kv_page_compact_launch", ret)
        _used_on(stream, rows, start, keep, offsets)
        return out[:n]

    def check(self) -> None:
        """Wait for the device and raise ValueError for what the calls since
        the last check() found wrong in their arguments."""
        torch.cuda.synchronize(self.device)     # calls on all streams
        bits = int(self.error.item())
        if bits:
            self.error.zero_()
            torch.cuda.synchronize(self.device)
            raise ValueError("page pool: " + "; ".join(text for bit, text in _ERRORS if bits & bit))


__all__ = ["PagePool", "OK", "NO_PAGES", "INVALID"]
