"""Rotary positions of new tokens: both pair layouts, part of the head, frequencies stretched for long contexts.

`rope_query` in attention.py is the one-token, whole-head, half-layout form whose fp32 angles agree bit for bit with the
key-reconstruction kernels.  `rotary_embedding` is for caches that hold rotated keys (dense or 8-bit): it turns queries
and keys of any number of tokens in one launch and reduces the angles in 64 bits, so that far positions keep their
accuracy.
"""
from __future__ import annotations

import math

import torch

from . import _C

__all__ = ["rotary_frequencies", "rotary_embedding"]


def rotary_frequencies(rotary_dim, theta=10000.0, *, scaling=None, factor=1.0, original_length=None, beta_fast=32.0,
                       beta_slow=1.0, low=1.0, high=4.0, device="cuda"):
    """Turning speed of each pair, for rotary_embedding: (inv_freq, magnitude) with inv_freq (rotary_dim / 2,) float64 on
    `device`, radians per position, and the factor on cosine and sine.  f_j = theta ** (-2 j / rotary_dim), then by
    `scaling` (factor = new context / original_length):

    None           f_j
    "linear"       f_j / factor (positions interpolated)
    "base"         theta * factor ** (d / (d - 2)) in place of theta: the slowest pair is slowed by `factor`, the fastest kept
    "wavelength"   f_j / factor for wavelengths over original_length / low, f_j for those below original_length / high,
                   in between the two blended by original_length / wavelength
    "yarn"         f_j / factor for pairs that turn less than beta_slow times over original_length, f_j for more than
                   beta_fast times, a linear ramp over the pair index in between; magnitude 0.1 ln(factor) + 1
    """
    dim = int(rotary_dim)
    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary_dim must be positive and even; got {rotary_dim}")
    if not theta > 0 or not factor >= 1.0:
        raise ValueError("theta must be positive and factor at least 1")
    if scaling in ("wavelength", "yarn") and not (original_length and original_length > 0):
        raise ValueError(f"scaling {scaling!r} needs original_length")
    magnitude = 1.0
    if scaling == "base":
        if dim == 2:
            raise ValueError("scaling 'base' needs rotary_dim > 2")
        theta = theta * factor ** (dim / (dim - 2))
    freq = [theta ** (-2.0 * j / dim) for j in range(dim // 2)]
    if scaling == "linear":
        freq = [f / factor for f in freq]
    elif scaling == "wavelength":
        if not high > low:
            raise ValueError("high must be above low")

        def blend(f):
            turns = original_length * f / (2 * math.pi)         # over the original context
            keep = min(max((turns - low) / (high - low), 0.0), 1.0)
            return f * keep + f / factor * (1.0 - keep)

        freq = [blend(f) for f in freq]
    elif scaling == "yarn":
        def pair_at(turns):                                      # the (fractional) pair that turns so often
            return dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(theta))

        first, last = max(math.floor(pair_at(beta_fast)), 0), min(math.ceil(pair_at(beta_slow)), dim - 1)
        ramp = [min(max((j - first) / max(last - first, 0.001), 0.0), 1.0) for j in range(dim // 2)]
        freq = [f / factor * r + f * (1.0 - r) for f, r in zip(freq, ramp)]
        magnitude = 0.1 * math.log(factor) + 1.0
    elif scaling not in (None, "base"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return torch.tensor(freq, dtype=torch.float64, device=device), magnitude


def rotary_embedding(query, key, inv_freq, position, *, interleaved=False, magnitude=1.0, out=None):
    """Turn queries and keys of new tokens to their positions; returns (query', key').

    query (bsz, num_heads, n, head_dim), key (bsz, num_kv_heads, n, head_dim) or None; inv_freq (rotary_dim / 2,) float64
    and `magnitude` from rotary_frequencies.  The first rotary_dim elements of every head are turned, as pairs (j, j +
    rotary_dim / 2) or, with `interleaved`, (2j, 2j + 1); the others are copied.  `position`: an int or an int32
    tensor (bsz,), the position of each sequence's first token with the others following it, or an int32 tensor (bsz,
    n) of every token's own (drafted trees).  `out`: a (query', key') pair to fill; it may be the inputs themselves, and share no memory with
    them otherwise."""
    shape = query.shape
    if len(shape) != 4:
        raise ValueError(f"query must be (bsz, num_heads, n, head_dim); got {tuple(shape)}")
    b, H, n, D = shape
    dt = query.dtype
    if key is None:
        idx, KVH = _C.device_index(query, inv_freq), 0
    else:
        idx = _C.device_index(query, key, inv_freq)
        kshape = key.shape
        if len(kshape) != 4 or kshape[0] != b or kshape[2] != n or kshape[3] != D:
            raise ValueError(f"key must be ({b}, num_kv_heads, {n}, {D}); got {tuple(kshape)}")
        if key.dtype != dt:
            raise ValueError("all tensors of one call must share a dtype")
        KVH = kshape[1]
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be a contiguous float64 tensor of shape (rotary_dim / 2,)")
    rot = 2 * inv_freq.numel()
    if not 0 < rot <= D:
        raise ValueError(f"inv_freq holds {rot // 2} pairs; head_dim {D} has room for {D // 2}")
    pos_ptr, pos_i, psb, pst = 0, 0, 0, 0
    if isinstance(position, torch.Tensor):
        _C.device_index(query, position)
        pshape = position.shape
        if position.dtype != torch.int32 or not (pshape == (b,) or pshape == (b, n)):
            raise ValueError("positions must be an int32 device tensor of shape (bsz,) or (bsz, n)")
        if len(pshape) == 2:
            position = position.contiguous()
            pst = 1 if n > 1 else 0
        psb = position.stride(0)
        pos_ptr = position.data_ptr()
    else:
        pos_i = int(position)
        if not -2 ** 31 <= pos_i < 2 ** 31:
            raise ValueError("position must fit 32 bits")
    q, qs = query, query.stride()
    if qs[3] != 1 and D != 1:
        q = query.contiguous()
        qs = q.stride()
    k, ks = key, (0, 0, 0, 0)
    if key is not None:
        ks = key.stride()
        if ks[3] != 1 and D != 1:
            k = key.contiguous()
            ks = k.stride()
    if out is None:
        qo = torch.empty_like(q)
        ko = None if k is None else torch.empty_like(k)
        if (qo.stride(3) != 1 and D != 1) or (ko is not None and ko.stride(3) != 1 and D != 1):
            qo = torch.empty(shape, dtype=dt, device=q.device)
            ko = None if k is None else torch.empty(k.shape, dtype=dt, device=q.device)
    else:
        qo, ko = out
        if (ko is None) != (key is None):
            raise ValueError("out must be a (query', key') pair like the inputs")
        for o, t in ((qo, query), (ko, key)):
            if o is None:
                continue
            _C.device_index(query, o)
            if o.shape != t.shape or o.dtype != dt or (o.stride(3) != 1 and D != 1):
                raise ValueError("outputs must have the inputs' shapes and dtype and a contiguous last dim")
            for size, a, c in zip(o.shape, o.stride(), t.stride()):
                if size > 1 and (a == 0 or (a != c and o.data_ptr() == t.data_ptr())):
                    raise ValueError("outputs must have an element of memory each, in place exactly the input's")
    if query.numel() == 0:
        if key is not None and key.numel():      # no query heads: the keys turn as the call's only heads
            rotary_embedding(key, None, inv_freq, position, interleaved=interleaved, magnitude=magnitude, out=(ko, None))
        return qo, ko
    qt, kt, kp, kop = qo.stride(), (0, 0, 0, 0), 0, 0
    if k is not None:
        kt, kp, kop = ko.stride(), k.data_ptr(), ko.data_ptr()
    _C.launch("xkv_rotary", _C.ROTARY_PARAMS.pack(
        _C.dtype_code(q), b, H, KVH, n, D, rot, 1 if interleaved else 0, pos_i, magnitude, pos_ptr, psb, pst,
        inv_freq.data_ptr(), q.data_ptr(), qs[0], qs[1], qs[2], kp, ks[0], ks[1], ks[2],
        qo.data_ptr(), qt[0], qt[1], qt[2], kop, kt[0], kt[1], kt[2]), idx)
    return qo, ko
