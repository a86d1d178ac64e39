"""Key / value caches held in 8 bits: one code per element and one fp32 scale per (token, KV head) row.

A step writes its new rows with `quantized_cache_append`, attends with `group_query_attention_quantized` (attention.py),
which reads the codes directly, and `quantized_cache_read` gives rows back dense.  With top the largest magnitude of a row
and C the largest code (127 for int8, 448 for e4m3): scale = top * (1 / C), code = round(x * (C * (1 / top))), value
= code * scale, so an int8 value is within half a step, top / 254, of what was written and an e4m3 one within 2^-4 of itself (or
2^-10 top / 448 near zero)."""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _C

__all__ = ["QuantizedCache", "quantized_cache", "quantized_cache_append", "quantized_cache_read"]

_CODE_DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


@dataclass
class QuantizedCache:
    """Codes (bsz, num_kv_heads, capacity, head_dim) int8 or float8_e4m3fn, innermost contiguous, and scales (bsz,
    num_kv_heads, capacity) float32, innermost contiguous.  Any tensors of these shapes do; strides are free elsewhere."""
    key_codes: torch.Tensor
    key_scales: torch.Tensor
    value_codes: torch.Tensor
    value_scales: torch.Tensor


def quantized_cache(batch, num_kv_heads, capacity, head_dim, *, code="int8", device="cuda"):
    """A cache of zeros.  `code`: "int8" or "e4m3"."""
    if code not in _CODE_DTYPES:
        raise ValueError(f"code must be one of {sorted(_CODE_DTYPES)}; got {code!r}")
    shape = (batch, num_kv_heads, capacity)
    codes = [torch.zeros((*shape, head_dim), dtype=torch.uint8, device=device).view(_CODE_DTYPES[code]) for _ in range(2)]
    scales = [torch.zeros(shape, dtype=torch.float32, device=device) for _ in range(2)]
    return QuantizedCache(codes[0], scales[0], codes[1], scales[1])


def check_cache(cache):
    """(device index, batch, num_kv_heads, capacity, head_dim, code) of a cache whose tensors fit together, and the
    strides of key_codes, value_codes, key_scales and value_scales; raises where they do not."""
    kc, ks, vc, vs = cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales
    idx = _C.device_index(kc, ks, vc, vs)
    code = _C.CACHE_CODES.get(kc.dtype)
    if code is None or vc.dtype != kc.dtype:
        raise ValueError(f"codes must be int8 or float8_e4m3fn, keys and values alike; got {kc.dtype} and {vc.dtype}")
    shape = kc.shape
    if len(shape) != 4 or vc.shape != shape:
        raise ValueError(f"codes must be (bsz, num_kv_heads, capacity, head_dim); got {tuple(kc.shape)} and {tuple(vc.shape)}")
    b, h, cap, d = shape
    if ks.dtype != torch.float32 or vs.dtype != torch.float32 or ks.shape != shape[:3] or vs.shape != shape[:3]:
        raise ValueError(f"scales must be float32 ({b}, {h}, {cap}) tensors")
    kcs, vcs, kss, vss = kc.stride(), vc.stride(), ks.stride(), vs.stride()
    if (d > 1 and (kcs[3] != 1 or vcs[3] != 1)) or (cap > 1 and (kss[2] != 1 or vss[2] != 1)):
        raise ValueError("codes and scales need a contiguous last dim")
    return (idx, b, h, cap, d, code), (kcs, vcs, kss, vss)


def _start(position, b, like):
    """(int, pointer) of a first row given as an int or an int32 (bsz,) device tensor."""
    if isinstance(position, torch.Tensor):
        _C.device_index(like, position)
        if position.dtype != torch.int32 or position.dim() != 1 or position.numel() != b or not position.is_contiguous():
            raise ValueError("positions must be a contiguous int32 device tensor of shape (bsz,)")
        return 0, position.data_ptr()
    p = int(position)
    if not -2 ** 31 <= p < 2 ** 31:
        raise ValueError("position must fit 32 bits")
    return p, 0


def _launch(entry, cache, dims, strides, n, dtype, pos, pos_ptr, len_ptr, k, a, v, c):
    idx, b, h, cap, d, code = dims
    kcs, vcs, kss, vss = strides
    _C.launch(entry, _C.CACHE_PARAMS.pack(
        dtype, code, b, h, n, cap, d, pos, pos_ptr, len_ptr, k.data_ptr(), a[0], a[1], a[2], v.data_ptr(), c[0], c[1], c[2],
        cache.key_codes.data_ptr(), kcs[0], kcs[1], kcs[2], cache.value_codes.data_ptr(), vcs[0], vcs[1], vcs[2],
        cache.key_scales.data_ptr(), kss[0], kss[1], cache.value_scales.data_ptr(), vss[0], vss[1]), idx)


def quantized_cache_append(cache, key, value, position, *, lengths=None):
    """Quantise new rows into the cache, in place; returns `cache`.

    key / value (bsz, num_kv_heads, n, head_dim), float32, bfloat16 or float16; `position` an int or an int32 device
    tensor (bsz,): the cache row of each sequence's first token, the others follow it.  `lengths` (int32 (bsz,)): only
    the first lengths[b] tokens of sequence b are written (padded prompts).  Rows outside the cache are left alone.  A
    row with an infinity or a NaN reads back as NaN throughout."""
    dims, strides = check_cache(cache)
    idx, b, h, cap, d, _ = dims
    _C.device_index(cache.key_codes, key, value)
    shape = key.shape
    if len(shape) != 4 or shape != value.shape or shape[0] != b or shape[1] != h or shape[3] != d:
        raise ValueError(f"key and value must be ({b}, {h}, n, {d}); got {tuple(key.shape)} and {tuple(value.shape)}")
    if key.dtype != value.dtype:
        raise ValueError("all tensors of one call must share a dtype")
    dtype = _C.dtype_code(key)
    pos, pos_ptr = _start(position, b, key)
    len_ptr = 0
    if lengths is not None:
        _C.device_index(key, lengths)
        if lengths.dtype != torch.int32 or tuple(lengths.shape) != (b,) or not lengths.is_contiguous():
            raise ValueError("lengths must be a contiguous int32 device tensor of shape (bsz,)")
        len_ptr = lengths.data_ptr()
    n = shape[2]
    if n == 0 or cap == 0 or b * h * d == 0:
        return cache
    k, v, a, c = key, value, key.stride(), value.stride()
    if a[3] != 1 and d != 1:
        k = key.contiguous()
        a = k.stride()
    if c[3] != 1 and d != 1:
        v = value.contiguous()
        c = v.stride()
    _launch("xkv_cache_append", cache, dims, strides, n, dtype, pos, pos_ptr, len_ptr, k, a, v, c)
    return cache


def quantized_cache_read(cache, position, length, *, dtype=torch.bfloat16):
    """Rows [position, position + length) of the cache as dense (key, value), each (bsz, num_kv_heads, length, head_dim)
    of `dtype`: code * scale, rounded once.  `position` as in quantized_cache_append; rows outside the cache are zeros."""
    dims, strides = check_cache(cache)
    idx, b, h, cap, d, _ = dims
    n = int(length)
    if not 0 <= n < 2 ** 31:
        raise ValueError("length must not be negative, and fit 32 bits")
    pos, pos_ptr = _start(position, b, cache.key_codes)
    k = torch.empty((b, h, n, d), dtype=dtype, device=cache.key_codes.device)
    v = torch.empty_like(k)
    code = _C.dtype_code(k)
    if n == 0 or b * h * d == 0:
        return k, v
    if cap == 0:
        return k.zero_(), v.zero_()
    a = (h * n * d, n * d, d)
    _launch("xkv_cache_read", cache, dims, strides, n, code, pos, pos_ptr, 0, k, a, v, a)
    return k, v
