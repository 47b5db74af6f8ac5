"""Pages of a block-paged cache: handed out, shared, copied, freed, compacted
(``dash_pages_*`` of libdash_b200.so).

A serving cache keeps K, V, index keys and k-bar rows of every layer in pages
with common ids.  :class:`CacheLayers` names those tensors once; every move of a
page runs over all of them in one launch.  :class:`PagePool` holds the tables on
the GPU: which pages a sequence owns, how many sequences hold a page, which
pages are free.  Nothing here waits for the GPU, and everything can be captured
into a CUDA graph; requests that do not fit leave their row as it was and are
recorded in the ``device_error`` word.  CUDA tensors only; every non-zero
library status raises.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Union

import torch

from . import _lib as L
from .ops import DeviceErrorWord, _need_cuda


def _call(fn: str, args, index: int) -> None:
    """Launch on the current stream of device ``index``, whatever the current
    device is."""
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _call(fn, args, index)
    rc = getattr(L.load(), fn)(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(index))
    if rc != L.DASH_OK:
        raise L.DashError(rc, L.last_error())


def _ints(t: Optional[torch.Tensor], name: str, index: int, n: Optional[int] = None) -> Optional[torch.Tensor]:
    """``t`` as a contiguous int32 vector (of ``n`` values) on CUDA device ``index``."""
    if t is None:
        return None
    if t.dtype is torch.int32 and t.get_device() == index and t.ndim == 1 and t.is_contiguous() and \
            (n is None or t.numel() == n):
        return t
    if t.get_device() != index:
        _need_cuda(t)
        raise ValueError(f"{name} is on {t.device}, not cuda:{index}")
    if t.dim() != 1 or (n is not None and t.shape[0] != n) or t.dtype not in _INTS:
        raise ValueError(f"{name} must be an int32 vector" + ("" if n is None else f" of {n} values"))
    return t.to(torch.int32).contiguous()


_INTS = (torch.int32, torch.int64)
_COPY = L.packer(L.DashPagesCopyArgs)
_PAGES = L.packer(L.DashPagesArgs, 2)             # behind the two pools


class CacheLayers:
    """The tensors of a paged cache, all indexed by the same page ids.

    Each is [num_pages, page_tokens, ...] with a contiguous entry per token (any
    stride between tokens and pages; [num_pages, 1, n] holds one entry per page,
    like k-bar rows).  Any dtype.  The handle keeps the tensors alive; build it
    once per set of caches."""

    def __init__(self, tensors: Sequence[torch.Tensor]):
        self.tensors = list(tensors)
        if not self.tensors:
            raise ValueError("a cache needs at least one tensor")
        first = self.tensors[0]
        self.device, self.num_pages = first.device, int(first.shape[0])
        self.index = first.get_device()
        self.c = (L.DashCacheTensor * len(self.tensors))()
        toks = set()
        for d, t in zip(self.c, self.tensors):
            _need_cuda(t)
            if t.device != self.device:
                raise ValueError("cache tensors must be on one device")
            if t.dim() < 2 or t.shape[0] != self.num_pages:
                raise ValueError(f"cache tensors must be [{self.num_pages}, page_tokens, ...], got {tuple(t.shape)}")
            e, inner = t.element_size(), 1
            for k in range(t.dim() - 1, 1, -1):
                if t.shape[k] != 1 and t.stride(k) != inner:
                    raise ValueError("a token's entry must be contiguous")
                inner *= t.shape[k]
            if inner * e > 1 << 30:
                raise ValueError("entries above 1 GiB are not supported")
            d.base, d.tok_bytes, d.page_toks = t.data_ptr(), inner * e, t.shape[1]
            d.tok_stride = inner * e if d.page_toks == 1 else t.stride(1) * e
            d.page_stride = t.stride(0) * e if self.num_pages > 1 else d.page_toks * d.tok_stride
            toks.add(int(d.page_toks))
        self.n, self.address = len(self.c), ctypes.addressof(self.c)
        # tokens per page, where all tensors agree
        self.page_tokens = toks.pop() if len(toks) == 1 else None


Layers = Union[CacheLayers, Sequence[torch.Tensor]]


def _layers(caches: Layers) -> CacheLayers:
    return caches if isinstance(caches, CacheLayers) else CacheLayers(caches)


def copy_pages(caches: Layers, src: torch.Tensor, dst: torch.Tensor,
               device_error: Optional[DeviceErrorWord] = None) -> None:
    """Page ``src[i]`` -> page ``dst[i]`` in every cache tensor (int32 vectors; a
    negative id skips the pair).  The pairs run at the same time: one whose
    destination is another pair's source or destination, or whose source is another
    pair's destination, is left out and recorded, as is one with an id past the
    last page."""
    layers = _layers(caches)
    src = _ints(src, "src", layers.index)
    n = src.numel()
    dst = _ints(dst, "dst", layers.index, n)
    if n:
        scratch = torch.empty(2 * n, dtype=torch.int32, device=layers.device)
        _call("dash_pages_copy", _COPY(layers.address, layers.n, n, src.data_ptr(), dst.data_ptr(), 0, scratch.data_ptr(),
                                       layers.num_pages, 1, 0, device_error.ptr if device_error is not None else 0),
              layers.index)


class PagePool:
    """Page tables of up to ``max_rows`` sequences over ``num_pages`` pages.

    ``block_table`` int32 [max_rows, max_blocks] (-1 behind a row's pages),
    ``n_blocks`` [max_rows], ``ref`` [num_pages] (rows holding the page),
    ``free_list`` [num_pages] (a stack, -1 behind its top), ``n_free`` [1]: CUDA
    tensors that the attention calls read directly."""

    def __init__(self, num_pages: int, max_rows: int, max_blocks: int, block_size: int, device="cuda"):
        i32 = dict(dtype=torch.int32, device=device)
        self._set(block_size, torch.zeros(num_pages, **i32),
                  torch.arange(num_pages - 1, -1, -1, **i32), torch.full((1,), num_pages, **i32),
                  torch.full((max_rows, max_blocks), -1, **i32), torch.zeros(max_rows, **i32))

    @classmethod
    def from_tensors(cls, *, block_size: int, ref, free_list, n_free, block_table, n_blocks) -> "PagePool":
        """A pool over existing tables (kept by reference)."""
        self = cls.__new__(cls)
        self._set(block_size, ref, free_list, n_free, block_table, n_blocks)
        return self

    def _set(self, block_size, ref, free_list, n_free, block_table, n_blocks):
        vecs = (ref, free_list, n_free, block_table, n_blocks)
        _need_cuda(*vecs)
        for t in vecs:
            if t.dtype != torch.int32 or t.device != ref.device or t.stride(-1) != 1:
                raise ValueError("pool tensors must be int32 on one device with unit inner stride")
        if block_table.dim() != 2 or free_list.shape != ref.shape or n_free.numel() != 1 or \
                n_blocks.shape != block_table.shape[:1]:
            raise ValueError("pool tensors do not fit one another")
        self.ref, self.free_list, self.n_free = ref, free_list, n_free
        self.block_table, self.n_blocks = block_table, n_blocks
        self.block_size, self.device, self.index = int(block_size), ref.device, ref.get_device()
        c = self.c = L.DashPagePool()
        c.ref, c.free_list, c.n_free = ref.data_ptr(), free_list.data_ptr(), n_free.data_ptr()
        c.block_table, c.bt_stride = block_table.data_ptr(), block_table.stride(0)
        c.n_blocks, c.num_pages = n_blocks.data_ptr(), ref.shape[0]
        c.max_rows, c.bt_width, c.block_size = block_table.shape[0], block_table.shape[1], self.block_size
        self.packed = bytes(c)

    def _args(self, device_error, rows=0, src=0, lens=0, n=0, layers=None, copy_src=0, copy_dst=0, n_moves=0,
              new_id=0, into=None) -> L.DashPagesArgs:
        return L.DashPagesArgs.from_buffer_copy(
            self.packed + (into or self).packed +
            _PAGES(rows, src, lens, n, *((0, 0) if layers is None else (layers.n, layers.address)), copy_src, copy_dst,
                   n_moves, new_id, device_error.ptr if device_error is not None else 0))

    def _own(self, caches: Layers) -> CacheLayers:
        layers = _layers(caches)
        if layers.device != self.device or layers.num_pages < self.c.num_pages:
            raise ValueError(f"the caches need {self.c.num_pages} pages on {self.device}")
        return layers

    def reserve(self, rows: torch.Tensor, lens: torch.Tensor,
                device_error: Optional[DeviceErrorWord] = None) -> None:
        """Row ``rows[i]`` gets pages for ``lens[i]`` tokens (it never loses any)."""
        rows = _ints(rows, "rows", self.index)
        n = rows.numel()
        lens = _ints(lens, "lens", self.index, n)
        _call("dash_pages_reserve", self._args(device_error, rows.data_ptr(), 0, lens.data_ptr(), n), self.index)

    def free(self, rows: torch.Tensor, keep: Optional[torch.Tensor] = None,
             device_error: Optional[DeviceErrorWord] = None) -> None:
        """Row ``rows[i]`` keeps its first ``keep[i]`` blocks (default none)."""
        rows = _ints(rows, "rows", self.index)
        n = rows.numel()
        keep = _ints(keep, "keep", self.index, n)
        _call("dash_pages_free", self._args(device_error, rows.data_ptr(), 0, 0 if keep is None else keep.data_ptr(), n),
              self.index)

    def fork(self, src: torch.Tensor, dst: torch.Tensor, lens: torch.Tensor, caches: Layers,
             device_error: Optional[DeviceErrorWord] = None) -> None:
        """The empty row ``dst[i]`` becomes a copy of the first ``lens[i]`` tokens
        of row ``src[i]``: full pages are shared, a partly filled last one is
        copied to a page of its own in every tensor of ``caches``.  Nothing is copied
        later: a row that goes back behind tokens of a shared page must not write
        there (fork it anew at the shorter length)."""
        layers = self._own(caches)
        src = _ints(src, "src", self.index)
        n = src.numel()
        dst, lens = _ints(dst, "dst", self.index, n), _ints(lens, "lens", self.index, n)
        if n == 0:
            return
        pairs = torch.empty(2 * n, dtype=torch.int32, device=self.device)
        at = pairs.data_ptr()
        _call("dash_pages_fork", self._args(device_error, dst.data_ptr(), src.data_ptr(), lens.data_ptr(), n, layers, at,
                                            at + 4 * n), self.index)

    def compact(self, caches: Layers, into: Optional["PagePool"] = None,
                device_error: Optional[DeviceErrorWord] = None,
                new_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Moves the held pages to the lowest ids.  With ``into`` (a pool of the
        same sizes) the new tables go there and this pool keeps the old ones,
        which stay usable until a page is handed out again: no page that they
        name is overwritten.  Whatever else is kept by page either is among
        ``caches`` or follows ``new_ids`` (int32 [num_pages]), which receives every
        page's new id (its own where it stays or is not held).  Returns the number of
        moved pages (int32 [1], on the GPU)."""
        layers, to = self._own(caches), self if into is None else into
        if to.device != self.device or to.block_size != self.block_size:
            raise ValueError("`into` must be a pool of the same device and block size")
        P = self.c.num_pages
        half = P // 2
        if new_ids is None:
            new_ids = torch.empty(P, dtype=torch.int32, device=self.device)
        elif new_ids.shape != (P,) or new_ids.dtype is not torch.int32 or new_ids.device != self.device or \
                not new_ids.is_contiguous():
            raise ValueError(f"new_ids must be contiguous int32 [{P}] on {self.device}")
        buf = torch.empty(2 * half + 1, dtype=torch.int32, device=self.device)
        at = buf.data_ptr()
        _call("dash_pages_compact", self._args(device_error, layers=layers, copy_src=at, copy_dst=at + 4 * half,
                                               new_id=new_ids.data_ptr(), n_moves=at + 8 * half, into=to), self.index)
        return buf[2 * half:]
