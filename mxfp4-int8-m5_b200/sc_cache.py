"""Calls of the key/value cache kernels: an INT8 cache that is quantized as it is written (host_model.QuantKVCache), attention of one or
several new rows to a bfloat16 or INT8 cache, and the move of accepted rows.  CUDA tensors of the current device, launched on torch's
current stream; there is no CPU path.

A cache is an object with k and v [hk, capacity, d] and `offset`, the positions that it holds: bfloat16 (host_model.KVCache), or int8 with
float32 scales ks and vs [hk, capacity], not negative.  Nothing here advances `offset`.

A call of few rows is shorter on the device than on the host: checks ask each tensor as little as they can."""
from array import array

import torch

from . import _lib

MAX_ROWS = 64           # new rows of one call: the bits of a mask
_BF16, _I8, _F32, _I32, _I64 = torch.bfloat16, torch.int8, torch.float32, torch.int32, torch.int64


def _tensors(cache):
    """(int8, keys, values, key scales, value scales, shape) of a cache; raises for a cache of any other form than the two."""
    k, v = cache.k, cache.v
    shape, dt = k.shape, k.dtype
    if v.dtype != dt or len(shape) != 3 or v.shape != shape:
        raise ValueError(f"cache of keys {tuple(shape)} {dt} and values {tuple(v.shape)} {v.dtype}: both [heads, capacity, d]")
    if dt == _BF16:
        _lib.require_here(k, v)
        return False, k, v, None, None, shape
    if dt != _I8:
        raise TypeError(f"cache of {dt}: bfloat16, or int8 with scales")
    ks, vs = cache.ks, cache.vs
    _lib.require_here(k, v, ks, vs)
    if ks.dtype != _F32 or vs.dtype != _F32 or ks.shape != shape[:2] or vs.shape != shape[:2]:
        raise ValueError(f"scales {tuple(ks.shape)} and {tuple(vs.shape)} of a cache {tuple(shape)}: float32 [heads, capacity]")
    return True, k, v, ks, vs, shape


def _strides(x, unit):
    """x [heads, rows, d] with a head and row stride that the kernels take (multiples of `unit` elements, unit column stride, aligned), and the strides."""
    hs, rs, cs = x.stride()
    H, L, d = x.shape
    if H == 1:
        hs = 0
    if L == 1:
        rs = 0
    if cs != 1 or hs % unit or rs % unit or x.data_ptr() % (2 * unit):
        return x.clone(memory_format=torch.contiguous_format), L * d, d      # (contiguous() keeps a view that starts off a boundary as it is)
    return x, hs, rs


def _position(cache, rows, capacity, pos_dev):
    """(host position, address of the device's or None) of the first new row."""
    if pos_dev is not None:
        _lib.require_here(pos_dev)
        if pos_dev.dtype != _I32 or pos_dev.numel() != 1:
            raise TypeError("a position on the device is one int32")
        return 0, pos_dev.data_ptr()
    pos = cache.offset
    if not 0 <= pos <= capacity - rows:
        raise ValueError(f"rows {pos} .. {pos + rows} of a cache of {capacity}")
    return pos, None


def kv_append(k, v, cache, pos_dev=None):
    """Keys and values of new tokens, bfloat16 [hk, L, d] of any strides, into rows offset .. (or pos_dev[0] ..: rows past the end are dropped) of
    an INT8 cache: s = amax / 127 per vector, code = rint(x (1 / s)).  A vector that is not finite reads back as NaN."""
    int8, kc, vc, ks, vs, (hk, cap, d) = _tensors(cache)
    if not int8:
        raise TypeError("kv_append quantizes into an int8 cache")
    shape = k.shape
    if k.dtype != _BF16 or v.dtype != _BF16 or len(shape) != 3 or v.shape != shape or shape[0] != hk or shape[2] != d:
        raise ValueError(f"keys {tuple(shape)} {k.dtype} and values {tuple(v.shape)} {v.dtype}: bfloat16 [{hk}, tokens, {d}]")
    _lib.require_here(k, v, contiguous=False)
    L = shape[1]
    pos, dev = _position(cache, L, cap, pos_dev)
    (k, khs, krs), (v, vhs, vrs) = _strides(k, 8), _strides(v, 8)
    _lib.call("scmx_kv_append", k.data_ptr(), khs, krs, v.data_ptr(), vhs, vrs, L, hk, d, pos, dev, cap, kc.data_ptr(), ks.data_ptr(), vc.data_ptr(),
              vs.data_ptr(), _lib.stream())


def kv_read(cache, start=0, end=None):
    """Rows start .. end (default: offset) of an INT8 cache as bfloat16 keys and values [hk, end - start, d]."""
    int8, kc, vc, ks, vs, (hk, cap, d) = _tensors(cache)
    if not int8:
        raise TypeError("kv_read reads an int8 cache; a bfloat16 cache's rows are its tensors'")
    end = cache.offset if end is None else end
    if not 0 <= start <= end <= cap:
        raise ValueError(f"rows {start} .. {end} of a cache of {cap}")
    k, v = ks.new_empty((2, hk, end - start, d), dtype=_BF16).unbind()
    _lib.call("scmx_kv_read", kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), start, end - start, hk, d, cap, k.data_ptr(), v.data_ptr(), _lib.stream())
    return k, v


def kv_keep(caches, rows, pos=None, pos_dev=None):
    """In every cache (of equal shape and type) row pos + rows[j] becomes row pos + j; pos defaults to the first cache's offset.  rows: int32 [n <= 64] on
    the device, n the rows that were written from pos on; negative entries leave their row, as verify_draft pads its list.  A cache is listed once."""
    _lib.require_here(rows)
    n = rows.numel()
    if rows.dtype != _I32 or not 1 <= n <= MAX_ROWS:
        raise ValueError(f"kv_keep: {n} rows of {rows.dtype}: int32, 1 .. {MAX_ROWS}")
    if not caches:
        return
    int8, _, _, _, _, shape = _tensors(caches[0])
    hk, cap, d = shape
    if pos_dev is not None:
        pos, dev = _position(None, n, cap, pos_dev)
    else:
        pos, dev = caches[0].offset if pos is None else pos, None
        if not 0 <= pos <= cap - n:
            raise ValueError(f"rows {pos} .. {pos + n} of a cache of {cap}")
    layers, here, dt = [], rows.get_device(), _I8 if int8 else _BF16
    for c in caches:                     # the checks of _tensors, for many layers
        k, v = c.k, c.v
        if k.dtype != dt or v.dtype != dt or k.shape != shape or v.shape != shape:
            raise ValueError("kv_keep: caches of one shape and type")
        if k.get_device() != here or v.get_device() != here or not (k.is_contiguous() and v.is_contiguous()):
            _lib.require_here(k, v)
        if int8:
            _tensors(c)
            layers += (k.data_ptr(), v.data_ptr(), c.ks.data_ptr(), c.vs.data_ptr())
        else:
            layers += (k.data_ptr(), v.data_ptr(), 0, 0)
    if len({*layers[::4], *layers[1::4]}) < 2 * len(caches):      # its rows would move twice, or while others move
        raise ValueError("kv_keep: a cache's tensors are in the list twice")
    table = array("Q", layers)
    _lib.call("scmx_kv_keep", table.buffer_info()[0], len(caches), rows.data_ptr(), n, pos, dev, hk, d, cap, int8, _lib.stream())


def attention_supported(hq, hk, d):
    return d in (64, 128) and hk > 0 and hq % hk == 0


def cache_attention(q, cache, scale, mask=None, pos_dev=None):
    """Attention of n <= 64 new rows, q bfloat16 [hq, n, d], to a cache that already holds their keys and values at rows offset .. offset + n - 1 (pos_dev[0] ..
    if given, so that a captured call can be replayed while the sequence grows; one outside the cache is taken as the nearest inside) -> bfloat16 [n, hq d].  Row i sees every position before
    them, and new row j if bit j of mask[i] is set (int64 [n], sc_draft.draft_mask; None: j <= i).  A row that sees nothing gives zeros."""
    int8, kc, vc, ks, vs, (hk, cap, d) = _tensors(cache)
    shape = q.shape
    if q.dtype != _BF16 or len(shape) != 3 or shape[2] != d or not attention_supported(shape[0], hk, d):
        raise ValueError(f"queries {tuple(shape)} {q.dtype} for a cache {(hk, cap, d)}: bfloat16 [a multiple of {hk}, rows, {d}], d 64 or 128")
    hq, n, _ = shape
    if not 1 <= n <= MAX_ROWS:
        raise ValueError(f"{n} rows (1 .. {MAX_ROWS})")
    _lib.require_here(q, contiguous=False)
    bits = None
    if mask is not None:
        _lib.require_here(mask)
        if mask.dtype != _I64 or mask.numel() != n:
            raise ValueError(f"mask {tuple(mask.shape)} {mask.dtype}: int64 [{n}]")
        bits = mask.data_ptr()
    pos, dev = _position(cache, n, cap, pos_dev)
    q, qhs, qrs = _strides(q, 4)
    out = q.new_empty((n, hq * d))
    size = _lib.lib().scmx_cache_attn_scratch(cap if dev else pos + n, n, hq, hk, d)
    scratch = q.new_empty(size // 2) if size else None       # this call's own: graphs may be replayed side by side
    _lib.call("scmx_cache_attn", q.data_ptr(), qhs, qrs, kc.data_ptr(), vc.data_ptr(), ks.data_ptr() if int8 else None, vs.data_ptr() if int8 else None, int8,
              bits, n, pos, dev, cap, hq, hk, d, scale, out.data_ptr(), scratch.data_ptr() if size else None, size, _lib.status_ptr(), _lib.stream())
    return out
