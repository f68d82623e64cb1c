"""Calls of the key/value cache kernels: an INT8 cache that is quantized as it is written (host_model.QuantKVCache), attention of one or
several new rows to a bfloat16 or INT8 cache, and the move of accepted rows.  CUDA tensors of the current device, launched on torch's
current stream; there is no CPU path.

A cache is an object with k and v [hk, capacity, d] and `offset`, the positions that it holds: bfloat16 (host_model.KVCache), or int8 with
float32 scales ks and vs [hk, capacity].  Nothing here advances `offset`."""
import torch

from . import _lib

MAX_ROWS = 64           # new rows of one call: the bits of a mask


def _is_int8(cache):
    """Whether a cache holds INT8 codes; raises for a cache of any other form than the two."""
    k, v = cache.k, cache.v
    int8 = k.dtype == torch.int8
    if v.dtype != k.dtype or not (int8 or k.dtype == torch.bfloat16):
        raise TypeError(f"cache of {k.dtype} keys and {v.dtype} values: bfloat16, or int8 with scales")
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError(f"cache of keys {tuple(k.shape)} and values {tuple(v.shape)}: both [heads, capacity, d]")
    tensors = (k, v, cache.ks, cache.vs) if int8 else (k, v)
    _lib.require_here(*tensors)
    if int8 and not (cache.ks.shape == cache.vs.shape == k.shape[:2] and cache.ks.dtype == cache.vs.dtype == torch.float32):
        raise ValueError(f"scales {tuple(cache.ks.shape)} and {tuple(cache.vs.shape)} of a cache {tuple(k.shape)}: float32 [heads, capacity]")
    return int8


def _strides(x, unit):
    """x [heads, rows, d] with a head and row stride that the kernels take (multiples of `unit` elements, unit column stride, aligned), and the strides."""
    H, L, d = x.shape
    hs, rs = (x.stride(0) if H > 1 else 0), (x.stride(1) if L > 1 else 0)
    if (x.stride(2) != 1 and d > 1) or hs % unit or rs % unit or x.data_ptr() % (2 * unit):
        x = x.contiguous()
        hs, rs = L * d, d
    return x, hs, rs


def _pos_dev(pos_dev):
    if pos_dev is not None:
        _lib.require_here(pos_dev)
        if pos_dev.dtype != torch.int32 or pos_dev.numel() != 1:
            raise TypeError("a position on the device is one int32")
    return _lib.ptr(pos_dev)


def kv_append(k, v, cache, pos_dev=None):
    """Keys and values of new tokens, bfloat16 [hk, L, d] of any strides, into rows offset .. (or pos_dev[0] ..: rows past the end are dropped) of
    an INT8 cache: s = amax / 127 per vector, code = rint(x (1 / s)).  A vector that is not finite reads back as NaN."""
    if not _is_int8(cache):
        raise TypeError("kv_append quantizes into an int8 cache")
    hk, cap, d = cache.k.shape
    if k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16 or k.dim() != 3 or k.shape != v.shape or k.shape[0] != hk or k.shape[2] != d:
        raise ValueError(f"keys {tuple(k.shape)} {k.dtype} and values {tuple(v.shape)} {v.dtype}: bfloat16 [{hk}, tokens, {d}]")
    _lib.require_here(k, v, contiguous=False)
    L = k.shape[1]
    if pos_dev is None and not 0 <= cache.offset <= cap - L:
        raise ValueError(f"rows {cache.offset} .. {cache.offset + L} of a cache of {cap}")
    (k, khs, krs), (v, vhs, vrs) = _strides(k, 8), _strides(v, 8)
    _lib.call("scmx_kv_append", k.data_ptr(), khs, krs, v.data_ptr(), vhs, vrs, L, hk, d, 0 if pos_dev is not None else cache.offset, _pos_dev(pos_dev), cap,
              cache.k.data_ptr(), cache.ks.data_ptr(), cache.v.data_ptr(), cache.vs.data_ptr(), _lib.stream())


def kv_read(cache, start=0, end=None):
    """Rows start .. end (default: offset) of an INT8 cache as bfloat16 keys and values [hk, end - start, d]."""
    if not _is_int8(cache):
        raise TypeError("kv_read reads an int8 cache; a bfloat16 cache's rows are its tensors'")
    hk, cap, d = cache.k.shape
    end = cache.offset if end is None else end
    if not 0 <= start <= end <= cap:
        raise ValueError(f"rows {start} .. {end} of a cache of {cap}")
    k, v = (torch.empty((hk, end - start, d), dtype=torch.bfloat16, device=cache.k.device) for _ in range(2))
    _lib.call("scmx_kv_read", cache.k.data_ptr(), cache.ks.data_ptr(), cache.v.data_ptr(), cache.vs.data_ptr(), start, end - start, hk, d, cap, k.data_ptr(),
              v.data_ptr(), _lib.stream())
    return k, v


def kv_keep(caches, rows, pos=None, pos_dev=None):
    """In every cache (of equal shape and type) row pos + rows[j] becomes row pos + j; pos defaults to the first cache's offset.  rows: int32 [n <= 64] on
    the device, n the rows that were written from pos on; negative entries leave their row, as verify_draft pads its list."""
    _lib.require_here(rows)
    n = rows.numel()
    if rows.dtype != torch.int32 or not 1 <= n <= MAX_ROWS:
        raise ValueError(f"kv_keep: {n} rows of {rows.dtype}: int32, 1 .. {MAX_ROWS}")
    if not caches:
        return
    int8, shape = _is_int8(caches[0]), caches[0].k.shape
    hk, cap, d = shape
    if any(_is_int8(c) != int8 or c.k.shape != shape for c in caches):
        raise ValueError("kv_keep: caches of one shape and type")
    pos = caches[0].offset if pos is None else pos
    if pos_dev is None and not 0 <= pos <= cap - n:
        raise ValueError(f"rows {pos} .. {pos + n} of a cache of {cap}")
    layers = (_lib.ScmxKvLayer * len(caches))()
    for ly, c in zip(layers, caches):
        ly.k, ly.v = c.k.data_ptr(), c.v.data_ptr()
        if int8:
            ly.ks, ly.vs = c.ks.data_ptr(), c.vs.data_ptr()
    _lib.call("scmx_kv_keep", layers, len(caches), rows.data_ptr(), n, pos, _pos_dev(pos_dev), hk, d, cap, int(int8), _lib.stream())


def attention_supported(hq, hk, d):
    return d in (64, 128) and hk > 0 and hq % hk == 0


def cache_attention(q, cache, scale, mask=None, pos_dev=None):
    """Attention of n <= 64 new rows, q bfloat16 [hq, n, d], to a cache that already holds their keys and values at rows offset .. offset + n - 1 (pos_dev[0] ..
    if given, so that a captured call can be replayed while the sequence grows) -> bfloat16 [n, hq d].  Row i sees every position before
    them, and new row j if bit j of mask[i] is set (int64 [n], sc_draft.draft_mask; None: j <= i).  A row that sees nothing gives zeros."""
    int8 = _is_int8(cache)
    hk, cap, d = cache.k.shape
    if q.dtype != torch.bfloat16 or q.dim() != 3 or q.shape[2] != d or not attention_supported(q.shape[0], hk, d):
        raise ValueError(f"queries {tuple(q.shape)} {q.dtype} for a cache {tuple(cache.k.shape)}: bfloat16 [a multiple of {hk}, rows, {d}], d 64 or 128")
    hq, n, _ = q.shape
    if not 1 <= n <= MAX_ROWS:
        raise ValueError(f"{n} rows (1 .. {MAX_ROWS})")
    _lib.require_here(q, contiguous=False)
    if mask is not None:
        _lib.require_here(mask)
        if mask.dtype != torch.int64 or mask.numel() != n:
            raise ValueError(f"mask {tuple(mask.shape)} {mask.dtype}: int64 [{n}]")
    pos = 0 if pos_dev is not None else cache.offset
    if not 0 <= pos <= cap - n:
        raise ValueError(f"rows {pos} .. {pos + n} of a cache of {cap}")
    q, qhs, qrs = _strides(q, 4)
    out = torch.empty((n, hq * d), dtype=torch.bfloat16, device=q.device)
    size = _lib.lib().scmx_cache_attn_scratch(cap if pos_dev is not None else pos + n, n, hq, hk, d)
    scratch = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None       # this call's own: graphs may be replayed side by side
    _lib.call("scmx_cache_attn", q.data_ptr(), qhs, qrs, cache.k.data_ptr(), cache.v.data_ptr(), cache.ks.data_ptr() if int8 else None,
              cache.vs.data_ptr() if int8 else None, int(int8), _lib.ptr(mask), n, pos, _pos_dev(pos_dev), cap, hq, hk, d, float(scale), out.data_ptr(),
              _lib.ptr(scratch), size, _lib.status_buffer().data_ptr(), _lib.stream())
    return out
