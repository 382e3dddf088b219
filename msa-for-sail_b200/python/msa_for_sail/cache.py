"""Operators around the attention call of a serving step: page tables, norm and rotation with the cache write, 4-bit caches.

* ``paged_kv_tables``: the flat page table, slots and positions of a step from the requests' lengths, on the GPU;
* ``rope_plan`` / ``qk_norm_rope``: per-head norm of queries and keys, rotary positions (one axis or several) and the write of keys
  and values into the paged cache, in one pass;
* ``kv_cache_append``: the write alone;
* ``allocate_kv4_cache`` / ``kv4_read``: a cache that holds 4 bits a value; ``fmha_sail`` takes it as ``k`` and ``v``.

None of them has an upstream counterpart (upstream starts at the attention call, api.py:1480-1848).  All of them enqueue on the
current stream of their tensors' device and read nothing back; what is allocated comes from torch's caching allocator, so
they can be captured into CUDA graphs.
"""
import contextlib
import ctypes
import math
from fractions import Fraction
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from ._lib import MSA_DT_BF16, MSA_DT_E4M3, MSA_DT_F32, MSA_DT_KV4

KV4_TILE = 128                          # tokens of a page
KV4_ROW_BYTES = 72                      # 64 bytes of codes and 8 scales


_status_ptr = None                      # of api.py, set when that is imported


def _stream():
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _on(device):
    """A context in which `device` is the current one."""
    return contextlib.nullcontext() if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _launch(device, fn, args, what):
    """`fn` on the current stream of `device`."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(ctypes.byref(args), torch._C._cuda_getCurrentRawStream(index))
        if rc:
            _lib.check(rc, what)
    else:
        with torch.cuda.device(device):
            _lib.check(fn(ctypes.byref(args), _stream()), what)


def _same_device(device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.get_device() != device.index:
            raise ValueError(f"{name} is on {t.device}, expected {device}")


# ----------------------------------------------------------------------------
# 4-bit cache
# ----------------------------------------------------------------------------

def allocate_kv4_cache(num_pages: int, num_kv_heads: int, page_size: int = 128, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys' and values' caches of 4 bits a value: two uint8 tensors ``[num_pages, num_kv_heads, 128, 72]``, zeros.

    The 9 216 bytes of one page and head are one tile: 128 rows of 64 bytes (two e2m1 codes a byte, the even element in the low half),
    then 128 rows of eight e4m3 scales, one for each 16 elements (so the last two dimensions are not rows of 72 bytes).  Views
    of a larger allocation serve as well where the tiles stay contiguous and start at multiples of 16 bytes."""
    if page_size != KV4_TILE:
        raise ValueError(f"a 4-bit cache has pages of {KV4_TILE} tokens, got page_size={page_size}")
    if num_pages < 0 or num_kv_heads < 1:
        raise ValueError(f"num_pages={num_pages} must not be negative, num_kv_heads={num_kv_heads} must be positive")
    device = torch.cuda.current_device() if device is None else device
    shape = (num_pages, num_kv_heads, KV4_TILE, KV4_ROW_BYTES)
    return torch.zeros(shape, dtype=torch.uint8, device=device), torch.zeros(shape, dtype=torch.uint8, device=device)


def _check_kv4(name, t, num_kv_heads=None):
    shape, stride = t.shape, t.stride()
    if t.dtype != torch.uint8 or len(shape) != 4 or shape[2] != KV4_TILE or shape[3] != KV4_ROW_BYTES:
        raise ValueError(f"{name}: a 4-bit cache is uint8 [pages, Hkv, {KV4_TILE}, {KV4_ROW_BYTES}], got {t.dtype} {tuple(shape)}")
    if stride[3] != 1 or stride[2] != KV4_ROW_BYTES:
        raise ValueError(f"{name}: the tile of a page and head of a 4-bit cache must be contiguous")
    if stride[0] % 16 or stride[1] % 16 or t.data_ptr() % 16:
        raise ValueError(f"{name}: the tiles of a 4-bit cache must start at multiples of 16 bytes")
    if num_kv_heads is not None and shape[1] != num_kv_heads:
        raise ValueError(f"{name} has {shape[1]} KV heads, expected {num_kv_heads}")
    return stride


def _read(cache, stride, index, out, whole_pages, num_used=0):
    rows, shape = index.shape[0], cache.shape
    if rows == 0:
        return out
    if shape[0] == 0:
        return out.zero_()
    dev = cache.device
    _launch(dev, _lib.lib.msa_kv4_read, _lib.kv4_read_args(
        cache.data_ptr(), out.data_ptr(), index.data_ptr(), _status_ptr(dev) or 0, num_used, stride[0], stride[1], rows, shape[1], shape[0],
        whole_pages), "msa_kv4_read")
    return out


def _check_index(name, t, device):
    if t.dim() != 1 or t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 vector, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != device.index:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def kv4_read(cache: torch.Tensor, slot_map: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of a 4-bit cache as bf16 ``[tokens, Hkv, 128]`` (exact: code times scale; a scale per head is not applied).

    ``slot_map``: int32, ``page * 128 + offset`` of each token; rows of a negative slot are zeros."""
    stride = _check_kv4("cache", cache)
    if not cache.is_cuda:
        raise RuntimeError("kv4_read needs CUDA tensors (there is no CPU path)")
    dev = cache.device
    _check_index("slot_map", slot_map, dev)
    shape = (slot_map.shape[0], cache.shape[1], 128)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=dev)
    else:
        _same_device(dev, out=out)
        if out.dtype != torch.bfloat16 or tuple(out.shape) != shape or not out.is_contiguous():
            raise ValueError(f"out must be contiguous bf16 {shape}, got {out.dtype} {tuple(out.shape)}")
    return _read(cache, stride, slot_map, out, 0)


def unpack_pages(cache, kv_indices, num_used=0):
    """Pages of a 4-bit cache as bf16 ``[len(kv_indices), Hkv, 128, 128]``, the nearest page for a number that is none.  ``num_used``:
    where the device has the number of entries that count (0: all do); the pages behind them are left as they were."""
    out = torch.empty(kv_indices.shape[0], cache.shape[1], KV4_TILE, 128, dtype=torch.bfloat16, device=cache.device)
    return _read(cache, cache.stride(), kv_indices, out, 1, num_used)


# ----------------------------------------------------------------------------
# norm, rotation, cache write
# ----------------------------------------------------------------------------

class RopePlan(dict):
    """Frequencies of a rotation, prepared by ``rope_plan``; pass it unchanged to ``qk_norm_rope``."""


def rope_plan(rotary_dim: int = 128, base: float = 10000.0, inv_freq: Optional[Union[torch.Tensor, Sequence[float]]] = None,
              sections: Optional[Sequence[int]] = None, interleaved: bool = False, device=None) -> RopePlan:
    """Frequencies of a rotary embedding over the first ``rotary_dim`` elements of a head (a multiple of 32, at most 128).

    ``inv_freq``: the angle per position of each of the ``rotary_dim / 2`` pairs (scaled variants bring their own); default
    ``base ** (-2 i / rotary_dim)``.  ``sections``: pairs of each position axis, in order (time, height, width of a video token:
    three numbers that add up to ``rotary_dim / 2``); default one axis.  ``interleaved``: pairs are neighbours (2 i, 2 i + 1)
    instead of (i, i + rotary_dim / 2).

    Frequencies are kept as 64-bit fractions of a turn, so angles are exact at any position."""
    if rotary_dim % 32 or not 0 < rotary_dim <= 128:
        raise ValueError(f"rotary_dim must be a multiple of 32 in (0, 128], got {rotary_dim}")
    pairs = rotary_dim // 2
    if inv_freq is None:
        inv_freq = [base ** (-2 * i / rotary_dim) for i in range(pairs)]
    else:
        inv_freq = inv_freq.detach().double().cpu().tolist() if isinstance(inv_freq, torch.Tensor) else [float(x) for x in inv_freq]
    if len(inv_freq) != pairs:
        raise ValueError(f"inv_freq must have rotary_dim / 2 = {pairs} entries, got {len(inv_freq)}")
    if not all(math.isfinite(f) for f in inv_freq):
        raise ValueError("inv_freq must be finite")
    sections = [pairs] if sections is None else [int(n) for n in sections]
    if sum(sections) != pairs or min(sections) < 0:
        raise ValueError(f"sections must add up to rotary_dim / 2 = {pairs}, got {sections}")
    turns = []
    for f in inv_freq:
        n = round(Fraction(f) / _TWO_PI * (1 << 64)) % (1 << 64)
        turns.append(n - (1 << 64) if n >= 1 << 63 else n)
    axis = [i for i, n in enumerate(sections) for _ in range(n)]
    device = torch.cuda.current_device() if device is None else device
    return RopePlan(rotary_dim=rotary_dim, interleaved=bool(interleaved), axes=len(sections),
                    turns=torch.tensor(turns, dtype=torch.int64, device=device), axis=torch.tensor(axis, dtype=torch.int32, device=device))


# 2 pi to 39 digits: a frequency in turns is then as exact as the frequency
_TWO_PI = Fraction(6283185307179586476925286766559005768394, 10 ** 39)


def _rows(name, t, heads, tokens, device, dtypes=(torch.bfloat16,)):
    """Checks of [tokens, heads, 128]; the strides of tokens and heads."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != 128 or (heads is not None and shape[1] != heads) or (tokens is not None and shape[0] != tokens):
        raise ValueError(f"{name} must be [{'tokens' if tokens is None else tokens}, {'heads' if heads is None else heads}, 128], got {tuple(shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    s0, s1, s2 = t.stride()
    if s2 != 1:
        raise ValueError(f"{name} head_dim must be contiguous")
    unit = 16 if t.dtype == torch.bfloat16 else 8
    if t.data_ptr() % unit or s0 % 8 or s1 % 8:
        raise ValueError(f"{name}: rows must start at multiples of {unit} bytes")
    if t.get_device() != device.index:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return s0, s1


def _weight(name, w, heads, device):
    if w is None:
        return 0, 0
    if w.get_device() != device.index:
        raise ValueError(f"{name} is on {w.device}, expected {device}")
    if w.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{name} must be float32 or bfloat16, got {w.dtype}")
    shape, stride = w.shape, w.stride()
    if shape != (128,) and shape != (heads, 128):
        raise ValueError(f"{name} must be [128] or [{heads}, 128], got {tuple(shape)}")
    if stride[-1] != 1 or (len(shape) == 2 and stride[0] % 8) or w.data_ptr() % 16:
        raise ValueError(f"{name}: rows must be contiguous and start at multiples of 16 bytes")
    return w.data_ptr(), stride[0] if len(shape) == 2 else 0


def _scale(name, x, heads, device):
    """A scale is a float, or an fp32 tensor with one value per KV head (it stays on the device)."""
    if x is None:
        return 1.0, 0
    if isinstance(x, torch.Tensor):
        if x.dtype != torch.float32 or x.numel() != heads or not x.is_contiguous():
            raise ValueError(f"{name} must be a float or a contiguous float32 tensor of {heads} values, got {x.dtype} {tuple(x.shape)}")
        if x.get_device() != device.index:
            raise ValueError(f"{name} is on {x.device}, expected {device}")
        return 1.0, x.data_ptr()
    return float(x), 0


_CACHE_DTYPES = {torch.bfloat16: MSA_DT_BF16, torch.float8_e4m3fn: MSA_DT_E4M3, torch.uint8: MSA_DT_KV4}


def _cache_strides(name, c, dtype, heads, page_size, device):
    """(pointer, strides of pages, heads, tokens) of one cache."""
    if c.get_device() != device.index:
        raise ValueError(f"{name} is on {c.device}, expected {device}")
    if dtype == MSA_DT_KV4:
        stride = _check_kv4(name, c, heads)
        return c.data_ptr(), stride[0], stride[1], 0
    shape, stride = c.shape, c.stride()
    if len(shape) != 4 or shape[3] != 128 or stride[3] != 1:
        raise ValueError(f"{name} must be [pages, Hkv, page, 128] or [pages, page, Hkv, 128], got {tuple(shape)}")
    unit = 16 if dtype == MSA_DT_BF16 else 8
    if c.data_ptr() % unit or stride[0] % 8 or stride[1] % 8 or stride[2] % 8:
        raise ValueError(f"{name}: rows must start at multiples of {unit} bytes")
    if shape[2] == page_size and shape[1] == heads:
        return c.data_ptr(), stride[0], stride[1], stride[2]
    if shape[1] == page_size and shape[2] == heads:
        return c.data_ptr(), stride[0], stride[2], stride[1]
    raise ValueError(f"{name} must hold pages of {page_size} tokens and {heads} KV heads, got {tuple(shape)}")


def _cache_args(k_cache, v_cache, heads, slot_map, tokens, page_size, k_scale, v_scale, device):
    """Checks of the caches of a call, which have one type, layout and page count; their type, strides and scales."""
    if slot_map is None:
        raise ValueError("a cache needs slot_map")
    _check_index("slot_map", slot_map, device)
    if slot_map.shape[0] != tokens:
        raise ValueError(f"slot_map must have {tokens} entries, got {slot_map.shape[0]}")
    if k_cache.dtype != v_cache.dtype or k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache and v_cache must be alike, got {k_cache.dtype} {tuple(k_cache.shape)} and {v_cache.dtype} {tuple(v_cache.shape)}")
    dtype = _CACHE_DTYPES.get(k_cache.dtype)
    if dtype is None:
        raise ValueError(f"a cache is bfloat16, float8_e4m3fn or uint8 (4 bits), got {k_cache.dtype}")
    if dtype == MSA_DT_KV4 and page_size != KV4_TILE:
        raise ValueError(f"a 4-bit cache has pages of {KV4_TILE} tokens, got page_size={page_size}")
    if page_size < 1:
        raise ValueError(f"page_size={page_size} must be positive")
    if k_cache.shape[0] < 1:
        raise ValueError("the cache has no pages")
    if k_cache.shape[0] * page_size > (1 << 31) - 1:
        raise ValueError("slots of a cache of more than 2^31 - 1 tokens do not fit int32")
    if dtype == MSA_DT_BF16 and (k_scale is not None or v_scale is not None):
        raise ValueError("k_scale and v_scale belong to a quantised cache")
    return (dtype, _cache_strides("k_cache", k_cache, dtype, heads, page_size, device), _cache_strides("v_cache", v_cache, dtype, heads, page_size, device),
            _scale("k_scale", k_scale, heads, device), _scale("v_scale", v_scale, heads, device))


_NO_CACHE = (MSA_DT_BF16, (0, 0, 0, 0), (0, 0, 0, 0), (1.0, 0), (1.0, 0))


def qk_norm_rope(
    q: torch.Tensor,
    k: torch.Tensor,
    positions: Optional[torch.Tensor],
    rope: Optional[RopePlan],
    *,
    v: Optional[torch.Tensor] = None,
    norm: bool = True,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    q_out: Optional[torch.Tensor] = None,
    k_out: Optional[torch.Tensor] = None,
    q_scale: Optional[float] = None,
    k_cache: Optional[torch.Tensor] = None,
    v_cache: Optional[torch.Tensor] = None,
    slot_map: Optional[torch.Tensor] = None,
    page_size: int = 128,
    k_scale=None,
    v_scale=None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Norm every query and key head, rotate them, and write keys and values into the paged cache, in one pass.

    ``q [T, Hq, 128]``, ``k [T, Hkv, 128]`` bf16, any strides whose rows start at multiples of 16 bytes (slices of a fused projection's
    output).  ``norm``: ``x / sqrt(mean(x^2) + eps) * weight`` over each head; weights ``[128]`` or one row per head, float32 or
    bf16.  ``rope`` (from ``rope_plan``, None: no rotation) turns the pairs of a head by ``positions``: int32 or int64, ``[T]``, or
    ``[axes, T]`` where the plan has several axes.

    Without caches returns ``(q, k)`` in bf16.  With ``k_cache``, ``v_cache`` and ``v`` the rows go to ``slot_map[t]`` (int32,
    ``page * page_size + offset``; a negative slot writes nothing; slots of one call are distinct) and the result is ``(q, None)``,
    or ``(q, k_out)`` where that is given.  Caches are bf16 or e4m3 (HND or NHD, as ``fmha_sail`` takes them) or 4-bit
    (``allocate_kv4_cache``); cached keys are computed in 64 bits and rounded to bf16 (by way of 32 bits) before they are quantised.
    ``k_scale`` / ``v_scale`` (quantised caches): what the attention call will multiply by, a float or one float32 value per KV head.
    ``q_out`` may be ``q`` (in place) or float8_e4m3fn (then ``q``, rounded to bf16, is divided by ``q_scale`` and stored)."""
    if not q.is_cuda:
        raise RuntimeError("qk_norm_rope needs CUDA tensors (there is no CPU path)")
    dev = q.device
    q_strides = _rows("q", q, None, None, dev)
    T, hq = q.shape[0], q.shape[1]
    k_strides = _rows("k", k, None, T, dev)
    hk = k.shape[1]
    if rope is not None:
        if positions is None:
            raise ValueError("a rotation needs positions")
        if positions.dtype != torch.int32 and positions.dtype != torch.int64:
            raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
        axes, shape = rope["axes"], positions.shape
        if shape != (axes, T) and not (axes == 1 and shape == (T,)):
            raise ValueError(f"positions must be [{axes}, {T}]" + (f" or [{T}]" if axes == 1 else "") + f", got {tuple(shape)}")
        pos_stride = positions.stride()
        if T > 1 and pos_stride[-1] != 1:
            raise ValueError("positions of one axis must be contiguous")
        turns, axis = rope["turns"], rope["axis"]
        if positions.get_device() != dev.index or turns.get_device() != dev.index:
            raise ValueError(f"positions are on {positions.device} and the rope plan is on {turns.device}, expected {dev}")
        pos = (positions.data_ptr(), turns.data_ptr(), axis.data_ptr(), pos_stride[0] if len(shape) == 2 else 0, rope["rotary_dim"],
               rope["interleaved"], positions.dtype == torch.int64)
    else:
        pos = (0, 0, 0, 0, 0, 0, 0)
    if (k_cache is None) != (v_cache is None) or (v_cache is None) != (v is None):
        raise ValueError("k_cache, v_cache and v go together")
    if k_cache is not None:
        v_strides = _rows("v", v, hk, T, dev)
        dtype, kc, vc, ks, vs = _cache_args(k_cache, v_cache, hk, slot_map, T, page_size, k_scale, v_scale, dev)
        v_ptr, slots, num_pages = v.data_ptr(), slot_map.data_ptr(), k_cache.shape[0]
    else:
        if k_scale is not None or v_scale is not None or slot_map is not None:
            raise ValueError("slot_map, k_scale and v_scale belong to a cache")
        dtype, kc, vc, ks, vs = _NO_CACHE
        v_ptr, v_strides, slots, num_pages = 0, (0, 0), 0, 0
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=torch.bfloat16, device=dev)
        qo_strides = (hq * 128, 128)
    else:
        qo_strides = _rows("q_out", q_out, hq, T, dev, (torch.bfloat16, torch.float8_e4m3fn))
    q8 = q_out.dtype == torch.float8_e4m3fn
    if q_scale is not None and not q8:
        raise ValueError("q_scale belongs to an e4m3 q_out")
    if k_out is None and k_cache is None:
        k_out = torch.empty(k.shape, dtype=torch.bfloat16, device=dev)
    ko_strides = _rows("k_out", k_out, hk, T, dev) if k_out is not None else (0, 0)
    if not norm and (q_weight is not None or k_weight is not None):
        raise ValueError("weights belong to the norm")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError(f"q_weight and k_weight must have one dtype, got {q_weight.dtype} and {k_weight.dtype}")
    qw, qw_stride = _weight("q_weight", q_weight, hq, dev)
    kw, kw_stride = _weight("k_weight", k_weight, hk, dev)
    w = q_weight if q_weight is not None else k_weight
    if T == 0:
        return q_out, k_out
    _launch(dev, _lib.lib.msa_norm_rope, _lib.norm_rope_args(
        q.data_ptr(), k.data_ptr(), v_ptr, qw, kw, pos[0], pos[1], pos[2], q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(),
        kc[0], vc[0], slots, ks[1], vs[1], _status_ptr(dev) or 0, pos[3], *q_strides, *k_strides, *v_strides, *qo_strides, *ko_strides, qw_stride,
        kw_stride, kc[1], kc[2], kc[3], vc[1], vc[2], vc[3], T, hq, hk, pos[4], pos[5], 1 if norm else 0,
        MSA_DT_BF16 if w is not None and w.dtype == torch.bfloat16 else MSA_DT_F32, MSA_DT_E4M3 if q8 else MSA_DT_BF16, dtype, pos[6],
        page_size if slots else 0, num_pages, eps, 1.0 if q_scale is None else q_scale, ks[0], vs[0]), "msa_norm_rope")
    return q_out, k_out


def kv_cache_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slot_map: torch.Tensor,
                    page_size: int = 128, k_scale=None, v_scale=None) -> None:
    """Write keys and values that are ready (``[T, Hkv, 128]`` bf16) into the paged cache at ``slot_map``; caches, slots and scales
    as in ``qk_norm_rope``."""
    if not k.is_cuda:
        raise RuntimeError("kv_cache_append needs CUDA tensors (there is no CPU path)")
    dev = k.device
    k_strides = _rows("k", k, None, None, dev)
    T, hk = k.shape[0], k.shape[1]
    v_strides = _rows("v", v, hk, T, dev)
    dtype, kc, vc, ks, vs = _cache_args(k_cache, v_cache, hk, slot_map, T, page_size, k_scale, v_scale, dev)
    if T == 0:
        return
    a = _lib.MsaNormRopeArgs()
    a.k, a.v, a.slot_map, a.status = k.data_ptr(), v.data_ptr(), slot_map.data_ptr(), _status_ptr(dev)
    a.k_stride_tok, a.k_stride_head = k_strides
    a.v_stride_tok, a.v_stride_head = v_strides
    a.k_cache, a.k_cache_stride_page, a.k_cache_stride_head, a.k_cache_stride_tok = kc
    a.v_cache, a.v_cache_stride_page, a.v_cache_stride_head, a.v_cache_stride_tok = vc
    (a.k_scale, a.k_scale_head), (a.v_scale, a.v_scale_head) = ks, vs
    a.cache_dtype, a.page_size, a.num_pages = dtype, page_size, k_cache.shape[0]
    a.tokens, a.num_kv_heads, a.weight_dtype = T, hk, MSA_DT_F32
    _launch(dev, _lib.lib.msa_norm_rope, a, "msa_norm_rope")


# ----------------------------------------------------------------------------
# page tables
# ----------------------------------------------------------------------------

class PageTables(dict):
    """Tensors of a step's paged cache, made by ``paged_kv_tables``."""


_TABLES = ("kv_indices", "kv_page_indptr", "slot_map", "positions", "num_missing", "num_held", "num_free")


def paged_kv_tables(
    qo_lens: torch.Tensor,
    kv_lens: torch.Tensor,
    block_table: torch.Tensor,
    num_held: Optional[torch.Tensor] = None,
    free_pages: Optional[torch.Tensor] = None,
    num_free: Optional[torch.Tensor] = None,
    *,
    max_total_q: int,
    max_total_pages: Optional[int] = None,
    page_size: int = 128,
    num_held_out: Optional[torch.Tensor] = None,
    num_free_out: Optional[torch.Tensor] = None,
    out: Optional[PageTables] = None,
) -> PageTables:
    """Page table, slots and positions of a step, built on the GPU from the requests' lengths (no host read, graph-safe).

    ``qo_lens`` / ``kv_lens``: int32 ``[B]``, the new tokens of each request and its keys with them (as ``fmha_sail_plan`` takes them).
    ``block_table``: int32 ``[B, width]``, the physical page of each logical page.  With ``num_held`` (int32 ``[B]``: entries of each
    row that are set), ``free_pages`` (int32, a stack) and ``num_free`` (int32 ``[1]``) the pages that new tokens need are taken
    from the top of the stack, in the order of the requests, and written into ``block_table``; without them the rows are complete.

    Returns ``kv_indices`` (``[max_total_pages]``, default ``B * width``; -1 behind the last page) and ``kv_page_indptr`` for the attention
    call, ``slot_map`` (``[max_total_q]``, -1 behind the last token) for the cache write, ``positions`` for the rotation, ``num_held``
    and ``num_free`` (the counts after this step; pass ``num_held_out=num_held, num_free_out=num_free`` to update in place) and
    ``num_missing``: pages and tokens that found no place.  Where that is not zero, missing pages are 0 in ``kv_indices``, places
    behind the end of a ``kv_indices`` that is too short read as its last page, the tokens' slots are -1, and tokens past
    ``max_total_q`` are in no sequence of a device-made plan with the same ``max_total_q``: nothing goes out of bounds, but attention
    over such a request means nothing.

    ``out``: a former result of the same sizes, whose tensors are written again (a captured step's fixed addresses)."""
    if not qo_lens.is_cuda:
        raise RuntimeError("paged_kv_tables needs CUDA tensors (there is no CPU path)")
    dev = qo_lens.device
    _check_index("qo_lens", qo_lens, dev)
    _check_index("kv_lens", kv_lens, dev)
    B = qo_lens.shape[0]
    if kv_lens.shape[0] != B:
        raise ValueError(f"qo_lens and kv_lens must have the same length, got {B} and {kv_lens.shape[0]}")
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or block_table.shape[0] != B or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise ValueError(f"block_table must be int32 [{B}, width] with contiguous rows, got {block_table.dtype} {tuple(block_table.shape)}")
    if B > 1 and block_table.stride(0) < block_table.shape[1]:
        raise ValueError("rows of block_table must not overlap")
    if not 1 <= page_size <= (1 << 31) - 1 or max_total_q < 0:
        raise ValueError(f"page_size={page_size} must be positive and fit int32, max_total_q={max_total_q} must not be negative")
    alloc = num_held is not None
    if alloc != (free_pages is not None) or alloc != (num_free is not None):
        raise ValueError("num_held, free_pages and num_free go together")
    if not alloc and (num_held_out is not None or num_free_out is not None):
        raise ValueError("num_held_out and num_free_out need num_held, free_pages and num_free")
    width = block_table.shape[1]
    total_pages = B * width if max_total_pages is None else int(max_total_pages)
    if total_pages < 0 or total_pages > (1 << 31) - 1 or max_total_q > (1 << 31) - 1:
        raise ValueError(f"max_total_pages={total_pages} and max_total_q={max_total_q} must fit int32")
    if alloc:
        for name, t, n in (("num_held", num_held, B), ("free_pages", free_pages, None), ("num_free", num_free, 1),
                           ("num_held_out", num_held_out, B), ("num_free_out", num_free_out, 1)):
            if t is None:
                continue
            _check_index(name, t, dev)
            if n is not None and t.shape[0] != n:
                raise ValueError(f"{name} must have {n} entries, got {t.shape[0]}")
    if block_table.get_device() != dev.index:
        raise ValueError(f"block_table is on {block_table.device}, expected {dev}")
    names, counts = (_TABLES, [total_pages, B + 1, max_total_q, max_total_q, 1, B, 1]) if alloc else (_TABLES[:5], [total_pages, B + 1, max_total_q, max_total_q, 1])
    given = {"num_held": num_held_out, "num_free": num_free_out} if num_held_out is not None or num_free_out is not None else {}
    if out is not None:
        for name, n in zip(names, counts):
            _check_index(f"out[{name!r}]", out[name], dev)
            if out[name].shape[0] != n:
                raise ValueError(f"out[{name!r}] must have {n} entries, got {out[name].shape[0]}")
        given = {**out, **{name: t for name, t in given.items() if t is not None}}
    ws_ints = (_lib.check(_lib.lib.msa_page_tables_workspace_bytes(B), "msa_page_tables_workspace_bytes") + 3) // 4
    # one allocation for the outputs and the scans
    if given:
        kept = {name: given[name] for name in names if given.get(name) is not None}
        fresh = [(name, n) for name, n in zip(names, counts) if name not in kept]
        counts = [n for _, n in fresh] + [ws_ints]
        parts = torch.empty(sum(counts), dtype=torch.int32, device=dev).split_with_sizes(counts)
        res = PageTables(zip([name for name, _ in fresh], parts), **kept)
    else:
        counts.append(ws_ints)
        parts = torch.empty(sum(counts), dtype=torch.int32, device=dev).split_with_sizes(counts)
        res = PageTables(zip(names, parts))
    held = (num_held.data_ptr(), free_pages.data_ptr(), num_free.data_ptr(), res["num_held"].data_ptr(), res["num_free"].data_ptr(),
            free_pages.shape[0]) if alloc else (0, 0, 0, 0, 0, 0)
    _launch(dev, _lib.lib.msa_page_tables, _lib.page_tables_args(
        qo_lens.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(), held[0], held[1], held[2], res["kv_indices"].data_ptr(),
        res["kv_page_indptr"].data_ptr(), res["slot_map"].data_ptr(), res["positions"].data_ptr(), held[3], held[4], res["num_missing"].data_ptr(),
        parts[-1].data_ptr(), block_table.stride(0) if B > 1 else width, B, width, page_size, max_total_q, total_pages, held[5]), "msa_page_tables")
    return res
