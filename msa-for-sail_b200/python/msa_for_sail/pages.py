"""Pages of a cache: copies, requests that share a prefix, pages given back, pages in use moved together.

* ``kv_pages_copy``: pages to other pages, in every cache of a model at once;
* ``kv_pages_fork``: rows of the block table that share the pages of another row (parallel samples, beams);
* ``kv_pages_free``: pages that the requests' lengths, or the window of their attention, no longer need;
* ``kv_pages_compact``: pages in use moved to the lowest places, so that the end of a pool is free.

They work on what ``paged_kv_tables`` works on: ``block_table`` (int32 ``[B, width]``), ``num_held`` (int32 ``[B]``, the entries of
each row that are set), the stack ``free_pages`` (int32) and ``num_free`` (int32 ``[1]``).  ``shares`` (int32 ``[pages]``, zeros at first) counts
the rows that hold a page beyond the first one, so that a page taken by ``paged_kv_tables`` needs no entry.  All of it is on the GPU and
updated in place on the current stream of its device; nothing is read back, so the calls can be captured into CUDA graphs.
No upstream counterpart (upstream starts at the attention call).
"""
import ctypes
import functools
import struct
from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _lib, cache
from .cache import KV4_ROW_BYTES, KV4_TILE, _check_index, _launch

_CACHE = struct.Struct("@QqqiiiI")


@functools.lru_cache(maxsize=256)
def _pieces(shape, stride, size, kv4, page_size, by_token):
    """Pieces of a page of a cache of this shape: (bytes from its start, page stride, stride of pieces, pieces, their bytes, bytes of a token), or
    None if they are not evenly spaced.  ``by_token``: a page may be copied up to a token."""
    if by_token and len(shape) == 4:
        if kv4 and shape[2:] == (KV4_TILE, KV4_ROW_BYTES) and stride[2:] == (KV4_ROW_BYTES, 1) and page_size == KV4_TILE:
            # a 4-bit cache: the codes of a page and head, then the scales
            codes = KV4_TILE * 64
            return [(0, stride[0], stride[1], shape[1], codes, 64), (codes, stride[0], stride[1], shape[1], KV4_TILE * 8, 8)]
        # (both dimensions as long as a page: either could be the tokens, the page is copied whole)
        hnd, nhd = shape[2] == page_size != shape[1], shape[1] == page_size != shape[2]
        if hnd and stride[2:] == (shape[3], 1):
            row = shape[3] * size
            return [(0, stride[0] * size, stride[1] * size, shape[1], page_size * row, row)]
        if nhd and stride[2:] == (shape[3], 1):
            row = shape[2] * shape[3] * size
            return [(0, stride[0] * size, stride[1] * size, page_size, row, -1)]
    # the innermost dimensions as far as they are contiguous; what is left has to be one step
    length, d = 1, len(shape) - 1
    while d > 0 and (shape[d] == 1 or stride[d] == length):
        length *= shape[d]
        d -= 1
    parts, step = 1, length
    if d > 0:
        parts, step = shape[d], stride[d]
        d -= 1
        while d > 0 and (shape[d] == 1 or stride[d] == parts * step):
            parts *= shape[d]
            d -= 1
        if d > 0:
            return None
    return [(0, stride[0] * size, step * size, parts, length * size, 0)]


def _cache_list(caches, num_pages, page_size, device, by_token=False):
    """(packed ``MsaPageCache``s, their number, pages)"""
    if isinstance(caches, torch.Tensor):
        caches = (caches,)
    packed, index, like = [], device.index, None
    for i, t in enumerate(caches):
        if t.get_device() != index:
            raise ValueError(f"caches[{i}] is on {t.device}, expected {device}")
        layout = t.shape, t.stride(), t.dtype
        if layout == like:                    # the caches of a model's layers are alike
            ptr = t.data_ptr()
            for off, rest in pieces:
                packed.append(pack(ptr + off, *rest))
            continue
        shape, stride, dtype = layout
        if not shape or (num_pages is not None and shape[0] != num_pages):
            raise ValueError(f"caches[{i}] must have {'pages' if num_pages is None else f'{num_pages} pages'} as its first dimension, got shape {tuple(shape)}")
        num_pages = shape[0]
        if 0 in shape:
            continue
        if num_pages > 1 and stride[0] == 0:
            raise ValueError(f"caches[{i}]: pages must not overlap")
        pieces = _pieces(shape, stride, dtype.itemsize, dtype is torch.uint8, page_size, by_token)
        if pieces is None:
            raise ValueError(f"caches[{i}]: a page must be one piece of memory or evenly spaced pieces, got shape {tuple(shape)}, strides {stride}")
        like, pack, ptr = layout, _CACHE.pack, t.data_ptr()
        pieces = [(off, (*rest, 0)) for off, *rest in pieces]
        for off, rest in pieces:
            packed.append(pack(ptr + off, *rest))
    return b"".join(packed), len(packed), num_pages


@functools.lru_cache(maxsize=256)
def _workspace(name, *sizes):
    """int32 entries of the workspace of a call of these sizes."""
    name = f"msa_pages_{name}_workspace_bytes"
    return _lib.check(getattr(_lib.lib, name)(*sizes), name) // 4


def _address(packed):
    """Where the bytes are, while `packed` lives."""
    return ctypes.cast(packed, ctypes.c_void_p).value


def _vector(name, t, n, device):
    _check_index(name, t, device)
    if n is not None and t.shape[0] != n:
        raise ValueError(f"{name} must have {n} entries, got {t.shape[0]}")


def _tables(block_table, page_size, rows, others):
    """Checks of what every call but the copy has: ``rows``, int32 with an entry for each row of ``block_table``, and ``others``, int32 of given
    lengths; (device, rows, width, stride)."""
    dev = block_table.device
    index = dev.index
    if dev.type != "cuda":
        raise RuntimeError("pages of a cache need CUDA tensors (there is no CPU path)")
    shape, stride, i32 = block_table.shape, block_table.stride(), torch.int32
    if len(shape) != 2 or block_table.dtype is not i32 or (shape[1] > 1 and stride[1] != 1):
        raise ValueError(f"block_table must be int32 [B, width] with contiguous rows, got {block_table.dtype} {tuple(shape)}")
    B, width = shape
    if B > 1 and stride[0] < width:
        raise ValueError("rows of block_table must not overlap")
    for name, t in rows.items():
        if t.dtype is not i32 or t.shape != (B,) or t.get_device() != index or not t.is_contiguous():
            _vector(name, t, B, dev)
    for name, (t, n) in others.items():
        if t.dtype is not i32 or t.dim() != 1 or t.get_device() != index or not t.is_contiguous() or (n is not None and t.shape[0] != n):
            _vector(name, t, n, dev)
    if not 1 <= page_size <= (1 << 31) - 1:
        raise ValueError(f"page_size={page_size} must be positive and fit int32")
    return dev, B, width, stride[0] if B > 1 else width


def kv_pages_copy(caches: Union[torch.Tensor, Sequence[torch.Tensor]], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every cache.

    ``caches``: tensors whose first dimension is the pages of one pool, of any type and layout (keys and values of all layers, 4-bit
    caches, scales), as long as a page is one piece of memory or evenly spaced pieces.  ``src``, ``dst``: int32 ``[n]`` on the GPU; an
    entry with a negative number (a list of fixed size) copies nothing, nor does one past the pool.  Entries are copied in any order: a page of
    ``dst`` is there once and is not in ``src``."""
    first = caches if isinstance(caches, torch.Tensor) else caches[0] if len(caches) else src
    dev = first.device
    if dev.type != "cuda":
        raise RuntimeError("kv_pages_copy needs CUDA tensors (there is no CPU path)")
    _vector("src", src, None, dev)
    _vector("dst", dst, src.shape[0], dev)
    packed, n, num_pages = _cache_list(caches, None, 1, dev)
    if n == 0 or src.shape[0] == 0:
        return
    _launch(dev, _lib.lib.msa_pages_copy, _lib.pages_copy_args(
        _address(packed), src.data_ptr(), dst.data_ptr(), cache._status_ptr(dev) or 0, n, src.shape[0], num_pages, 1), "msa_pages_copy")


def kv_pages_fork(block_table: torch.Tensor, num_held: torch.Tensor, kv_lens: torch.Tensor, parents: torch.Tensor, children: torch.Tensor,
                  free_pages: torch.Tensor, num_free: torch.Tensor, shares: torch.Tensor,
                  caches: Union[torch.Tensor, Sequence[torch.Tensor]] = (), page_size: int = 128) -> torch.Tensor:
    """Make row ``children[i]`` a fork of row ``parents[i]``: a request with the same first ``kv_lens[parent]`` tokens.

    Full pages are shared (``shares`` + 1 each); the last page, where it is partly filled, is taken from the stack, in the order of the entries, and
    the used part is copied in every one of ``caches``: 4-bit caches, and tensors of any type with four dimensions that are taken as ``[pages, Hkv, page, D]``
    if the third is ``page_size``, as ``[pages, page, Hkv, D]`` if the second is.  Of other tensors with pages as the first dimension, and where both
    are, the whole page is copied; one with four dimensions and such a length that means something else (keys with the tokens last, say) is given as
    a view, ``t.flatten(1)``.  So whoever writes next writes into a page of its
    own, as long as neither row is cut back into a page that they share (``kv_pages_free`` with ``caches`` sees to that).  ``num_held`` and ``kv_lens``
    (int32 ``[B]``) of the child are set.

    ``parents``, ``children``: int32 ``[n]``; an entry with a negative number does nothing (a list of fixed size).  A row may be the parent of many.
    A child holds nothing before (``kv_pages_free`` it first).  Returns ``num_missing`` (int32 ``[1]``): entries that were not made, since a row is
    not in the table, is its own parent, holds pages already or is a child for the second time, and children that found no page on the
    stack for their last tokens, which end with their last full page (``kv_lens`` says where)."""
    n = parents.numel()
    dev, B, width, stride = _tables(block_table, page_size, {"num_held": num_held, "kv_lens": kv_lens}, {
        "parents": (parents, n), "children": (children, n), "free_pages": (free_pages, None), "num_free": (num_free, 1), "shares": (shares, None)})
    packed, num, pages = _cache_list(caches, shares.shape[0], page_size, dev, True)
    buf = torch.empty(_workspace("fork", B, n) + 1, dtype=torch.int32, device=dev)
    ptr = buf.data_ptr()
    _launch(dev, _lib.lib.msa_pages_fork, _lib.pages_fork_args(
        _address(packed), block_table.data_ptr(), num_held.data_ptr(), kv_lens.data_ptr(), parents.data_ptr(), children.data_ptr(),
        free_pages.data_ptr(), num_free.data_ptr(), shares.data_ptr(), ptr, ptr + 4, stride, num, n, pages, page_size, B, width, free_pages.shape[0]),
        "msa_pages_fork")
    return buf[:1]


def kv_pages_free(block_table: torch.Tensor, num_held: torch.Tensor, kv_lens: torch.Tensor, free_pages: torch.Tensor, num_free: torch.Tensor,
                  shares: Optional[torch.Tensor] = None, *, window_size: int = -1, num_sink_tokens: int = 0, page_size: int = 128,
                  caches: Union[torch.Tensor, Sequence[torch.Tensor]] = (), num_shared: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Give back the pages that no request needs any more.

    Row ``b`` keeps the pages of its first ``kv_lens[b]`` tokens: 0 for a request that ended, less than before where drafted tokens were
    rejected.  With ``window_size`` and ``num_sink_tokens`` (as ``fmha_sail_plan`` takes them) it keeps of those only what a query at place
    ``kv_lens[b]`` or later sees: call it with the length before the new tokens of a step, or after the attention over them.  (Without a window
    it sees all of them, sinks or not.)  Entries given back
    become -1 (``paged_kv_tables`` turns those into page 0, which a windowed call does not read) and ``num_held`` the number of pages of
    the length.

    A page of several rows (``shares``) loses a share for each and goes onto the stack with the last; without ``shares`` each page is in one row.
    Pages are pushed in the order of the rows and their entries.  Returns ``num_freed`` (int32 ``[1]``): how many were pushed.  ``free_pages`` has
    room for every page of the pool.

    A row that is cut back *into* a page it shares (below the length it was forked at, or its fork's) would write its next token into the other rows'
    page.  With ``caches`` (all of them, as ``kv_pages_fork`` takes them) such a row gets a page of its own from the stack, in the order of the rows, with
    a copy of its tokens, and gives up its share; of rows that are all cut back into one page the last keeps it.  ``num_shared`` (int32 ``[1]``, set
    here) counts the rows that are left with such a page: all of them without ``caches``, with them those that found the stack empty.  They must not be
    written to."""
    others = {"free_pages": (free_pages, None), "num_free": (num_free, 1)}
    if shares is not None:
        others["shares"] = (shares, None)
    if num_shared is not None:
        others["num_shared"] = (num_shared, 1)
    dev, B, width, stride = _tables(block_table, page_size, {"num_held": num_held, "kv_lens": kv_lens}, others)
    window = -1 if window_size is None else int(window_size)
    if window == 0 or window < -1 or window > (1 << 31) - 1:
        raise ValueError(f"window_size must be -1 (no window) or from 1 to 2^31 - 1, got {window_size}")
    if not 0 <= num_sink_tokens <= (1 << 31) - 1:
        raise ValueError(f"num_sink_tokens must be from 0 to 2^31 - 1, got {num_sink_tokens}")
    packed, num = b"", 0
    if num_shared is not None or len(caches):
        if shares is None:
            raise ValueError("caches and num_shared need shares: without them each page is in one row")
        packed, num, _ = _cache_list(caches, shares.shape[0], page_size, dev, True)
    buf = torch.empty(_workspace("free", B, width) + 1, dtype=torch.int32, device=dev)
    ptr = buf.data_ptr()
    _launch(dev, _lib.lib.msa_pages_free, _lib.pages_free_args(
        _address(packed) if num else 0, block_table.data_ptr(), num_held.data_ptr(), kv_lens.data_ptr(), free_pages.data_ptr(), num_free.data_ptr(),
        0 if shares is None else shares.data_ptr(), ptr, 0 if num_shared is None else num_shared.data_ptr(), ptr + 4, stride, num, B, width, page_size,
        free_pages.shape[0], (1 << 31) - 1 if shares is None else shares.shape[0], max(window, 0),
        int(num_sink_tokens) if window > 0 else 0), "msa_pages_free")
    return buf[:1]


class PageMoves(NamedTuple):
    """Moves of ``kv_pages_compact``: page ``src[i]`` is now page ``dst[i]`` for ``i < num_moved``; -1 behind them, so that
    ``kv_pages_copy`` takes the lists for further tensors."""
    src: torch.Tensor
    dst: torch.Tensor
    num_moved: torch.Tensor


def kv_pages_compact(block_table: torch.Tensor, num_held: torch.Tensor, free_pages: torch.Tensor, num_free: torch.Tensor,
                     caches: Union[torch.Tensor, Sequence[torch.Tensor]] = (), shares: Optional[torch.Tensor] = None,
                     *, num_pages: Optional[int] = None) -> PageMoves:
    """Move the pages in use to the lowest places, so that the free ones are the highest of the pool.

    In use are the pages in the rows of ``block_table`` (below ``num_held``), free are those on the stack; pages that are neither (one that is
    kept for padding, say) stay where they are.  Of the pages in use above the line, the lowest goes to the lowest free place below it, and so on.
    ``block_table``, ``shares`` and the pages of all ``caches`` (as in ``kv_pages_copy``) follow, and the stack is made anew, the lowest page on top.
    The pool has ``num_pages`` pages, by default as many as the caches or ``shares``.  Tables made before (``kv_indices``, slots) are void."""
    others = {"free_pages": (free_pages, None), "num_free": (num_free, 1)}
    if shares is not None:
        others["shares"] = (shares, num_pages)
    dev, B, width, stride = _tables(block_table, 1, {"num_held": num_held}, others)
    if shares is not None:
        num_pages = shares.shape[0]
    packed, num, num_pages = _cache_list(caches, num_pages, 1, dev)
    if num_pages is None or not 0 <= num_pages <= (1 << 31) - 1:
        raise ValueError("num_pages is needed where there are neither caches nor shares" if num_pages is None else f"num_pages={num_pages} must fit int32")
    ws = _workspace("compact", num_pages)
    src, dst, num_moved, ws = torch.empty(2 * num_pages + 1 + ws, dtype=torch.int32, device=dev).split_with_sizes([num_pages, num_pages, 1, ws])
    _launch(dev, _lib.lib.msa_pages_compact, _lib.pages_compact_args(
        _address(packed), block_table.data_ptr(), num_held.data_ptr(), free_pages.data_ptr(), num_free.data_ptr(),
        0 if shares is None else shares.data_ptr(), src.data_ptr(), dst.data_ptr(), num_moved.data_ptr(), ws.data_ptr(), stride, num, num_pages, 1, B, width,
        free_pages.shape[0]), "msa_pages_compact")
    return PageMoves(src, dst, num_moved)
