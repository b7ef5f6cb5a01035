"""Rotary position embedding of a layer's new rows fused with the cache update.

Drop-in for the two steps the reference's patched Qwen2 attention takes
between the projections and the attention call
(hsd/dots_ocr_pipeline/modeling_dots_ocr_hsd.py D:337-351):
``apply_rotary_pos_emb(query_states, key_states, cos, sin)`` and
``past_key_value.update(key_states, value_states, ...)`` (a ``torch.cat`` of
the whole layer cache).  One launch rotates the query rows in place in the
``q_proj`` output and writes the rotated key rows and the value rows into
preallocated cache planes; results are bit-identical to torch's bf16 ops.

:func:`rope_append_axes` does the same for positions with several axes (image
and video tokens; the HunYuan pipeline's four, H:2033), computing the angles
from the position ids instead of reading tables.
"""
from __future__ import annotations

import math
from fractions import Fraction

import torch

from . import _native as N


def _rows(t, name, width=None):
    t2 = t.reshape(-1, t.shape[-1]) if t.dim() != 2 else t
    if t2.dtype != torch.bfloat16 or not t2.is_cuda:
        raise TypeError(f"rope_append: {name} must be a bf16 CUDA tensor")
    if t2.stride(-1) != 1:
        raise ValueError(f"rope_append: {name} rows must be contiguous")
    if width is not None and t2.shape[-1] != width:
        raise ValueError(f"rope_append: {name} has {t2.shape[-1]} columns, expected {width}")
    return t2


def _cache(c, name):
    c3 = c.reshape(-1, c.shape[-2], c.shape[-1]) if c.dim() != 3 else c
    if c3.dtype != torch.bfloat16 or c3.shape[-1] != 128 or c3.stride(-1) != 1:
        raise ValueError(f"rope_append: {name} must be bf16 [..., Hkv, KV, 128] with contiguous rows")
    return c3


def rope_append(q, k, v, cos, sin, k_cache, v_cache, dst_row0, num_q_heads=None,
                num_kv_heads=None):
    """Rotate ``q`` in place and append rotated ``k`` and ``v`` to the caches.

    q: ``[..., Q, Hq * 128]`` (the ``q_proj`` output; may be a column slice of
    a fused projection) or None; k, v: ``[..., Q, Hkv * 128]``; cos, sin:
    ``[..., Q, 128]`` bf16 (the model's ``position_embeddings``); k_cache,
    v_cache: ``[..., Hkv, KV, 128]`` bf16, rows ``[dst_row0, dst_row0 + Q)``
    receive the new rows.  Returns the rotated queries as a
    ``[1, Hq, Q, 128]`` view (the reference's ``query_states`` layout), or
    None when q is None.  Asynchronous on the current stream.
    """
    kc, vc = _cache(k_cache, "k_cache"), _cache(v_cache, "v_cache")
    hkv = num_kv_heads or kc.shape[0]
    k2, v2 = _rows(k, "k", hkv * 128), _rows(v, "v", hkv * 128)
    n = k2.shape[0]
    if k2.stride(0) != v2.stride(0):
        raise ValueError("rope_append: k and v must share a row stride")
    c2, s2 = _rows(cos, "cos", 128), _rows(sin, "sin", 128)
    if c2.stride(0) != s2.stride(0) or c2.shape[0] != n or v2.shape[0] != n:
        raise ValueError("rope_append: cos / sin / k / v row counts or strides differ")
    if kc.stride() != vc.stride() or kc.shape != vc.shape or kc.shape[0] != hkv:
        raise ValueError("rope_append: k_cache and v_cache must have one layout")
    if dst_row0 < 0 or dst_row0 + n > kc.shape[1]:
        raise ValueError(f"rope_append: rows {dst_row0}..{dst_row0 + n} past the cache")
    hq, q2, qptr, qstride = 0, None, None, 0
    if q is not None:
        hq = num_q_heads or q.shape[-1] // 128
        q2 = _rows(q, "q", hq * 128)
        if q2.shape[0] != n:
            raise ValueError("rope_append: q and k row counts differ")
        qptr, qstride = N.ptr(q2), q2.stride(0)
    lib = N.load()
    N.check(lib.hsd_rope_append(qptr, qstride, N.ptr(k2), N.ptr(v2), k2.stride(0), N.ptr(c2),
                                N.ptr(s2), c2.stride(0), n, hq, hkv, 128, N.ptr(kc),
                                kc.stride(0), N.ptr(vc), vc.stride(0), kc.stride(1), dst_row0,
                                N.stream_handle()), "hsd_rope_append")
    if q2 is None:
        return None
    return q2.unflatten(-1, (hq, 128)).unsqueeze(0).transpose(1, 2)


# ---------------------------------------------------------------- several axes
# 2 pi to 240 bits, as a fraction (the first digits of pi are public constants)
_TWO_PI = Fraction("6.283185307179586476925286766559005768394338798750211641949889184615632812572"
                   "417997256069650684234136")
_MAX_AXES = 8


class RotaryAxes:
    """Frequencies of a rotary embedding whose 64 dimension pairs turn with
    several position axes (time / height / width, or the four axes of the
    HunYuan pipeline's ``[1, 4, Q]`` position ids, H:2033).

    ``sections[a]``: how many pairs turn with axis ``a``; they sum to 64.  By
    default the pairs are shared out in order (the first ``sections[0]`` pairs
    turn with axis 0, and so on); with ``interleaved`` pair ``i`` turns with
    axis ``i % A`` while ``i < A * sections[i % A]`` and with axis 0 beyond
    (the later axes then need an equal share at most ``64 // A`` each).
    ``theta``: pair ``i`` turns ``theta ** (-i / 64)`` rad per position, or
    ``inv_freq`` gives the 64 frequencies (a model's buffer: its exact values
    are used).  ``scaling`` multiplies the cosines and sines.

    The device tables are made here, once; one object serves every layer.
    """

    def __init__(self, sections, theta=1e6, interleaved=False, inv_freq=None, scaling=1.0,
                 device="cuda"):
        self.sections = [int(n) for n in sections]
        self.scaling = float(scaling)
        self.axes = axes = len(self.sections)
        if not 1 <= axes <= _MAX_AXES or min(self.sections) < 0 or sum(self.sections) != 64:
            raise ValueError(f"RotaryAxes: sections {self.sections} must be 1 to {_MAX_AXES} "
                             "counts that sum to 64 pairs")
        if interleaved:
            axis = [i % axes if i < axes * self.sections[i % axes] else 0 for i in range(64)]
            if [axis.count(a) for a in range(axes)] != self.sections:
                raise ValueError(f"RotaryAxes: sections {self.sections} cannot be interleaved")
        else:
            axis = [a for a, n in enumerate(self.sections) for _ in range(n)]
        if inv_freq is None:
            if not (math.isfinite(theta) and theta > 0):
                raise ValueError(f"RotaryAxes: theta {theta} must be positive")
            freq = [float(theta) ** (-i / 64) for i in range(64)]
        else:
            freq = torch.as_tensor(inv_freq, dtype=torch.float64).reshape(-1).tolist()
        if len(freq) != 64 or not all(math.isfinite(f) for f in freq):
            raise ValueError("RotaryAxes: 64 finite frequencies are needed")
        if not math.isfinite(self.scaling):
            raise ValueError("RotaryAxes: scaling must be finite")
        # turns per position in units of 2^-64 turn, modulo one turn
        turns = [round(Fraction(f) / _TWO_PI * 2 ** 64) % 2 ** 64 for f in freq]
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns],
                                  dtype=torch.int64, device=device)
        self.pair_axis = torch.tensor(axis, dtype=torch.int32, device=device)


def rope_append_axes(q, k, v, positions, rotary, k_cache, v_cache, dst_row0, out=None,
                     num_q_heads=None, num_kv_heads=None, status=None):
    """:func:`rope_append` for positions with several axes, without cos / sin
    tables: the angles come from the integer ``positions``.

    q, k, v, k_cache, v_cache, dst_row0 as in :func:`rope_append` (k and v may
    have different row strides); positions: int64 ``[A, Q]`` (``[1, A, Q]`` and
    ``[A, 1, Q]`` too; any strides, an expanded row included);
    rotary: the :class:`RotaryAxes` of the model.  The queries are rotated in
    place, or into ``out`` (``[..., Q, Hq * 128]`` bf16, not overlapping q).
    Arithmetic is fp32 with one rounding to bf16 (:func:`rope_append` reproduces
    torch's bf16 products); angles are off by 2^-25 half turns, that of fp32, up to
    positions of 2^39, and by ``|position| * 2**-64`` half turns beyond.
    Returns the rotated queries as a ``[1, Hq, Q, 128]`` view, or None when q
    is None.  Asynchronous on the device's current stream.

    A model that normalises queries and keys per head after the rotation (the
    HunYuan decoder) does so on the returned view and, in place, on the rows
    written to ``k_cache``; nothing is normalised here.
    """
    return N.ops().rope_append_axes(q, k, v, positions, rotary.turns, rotary.pair_axis,
                                    rotary.axes, rotary.scaling, k_cache, v_cache, dst_row0, out,
                                    num_q_heads, num_kv_heads, status)
