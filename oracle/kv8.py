"""8-bit cache oracle: sealing, unsealing and the values a sealed row stands for."""
from __future__ import annotations

import numpy as np
import torch

BLOCK = 64
MIN_AMAX = 2.0 ** -100


def seal(x):
    """bf16 / float ``[..., rows, 128]`` (rows a multiple of 64) -> (int8 of
    the same shape, float64 scales ``[..., rows // 64]``), in 64 bits:
    n = 127 x / a to the nearest, ties to even."""
    a = torch.as_tensor(x).double().numpy()
    lead, rows = a.shape[:-2], a.shape[-2]
    b = a.reshape(*lead, rows // BLOCK, BLOCK * a.shape[-1])
    fin = np.where(np.isfinite(b), np.abs(b), 0.0)
    amax = np.maximum(fin.max(-1), MIN_AMAX)
    t = np.where(np.isnan(b), 0.0, np.clip(b, -amax[..., None], amax[..., None]))
    n = np.rint(127 * t / amax[..., None])
    return n.reshape(a.shape).astype(np.int8), amax / 127


def values(data, scale):
    """float64 values of sealed rows, with the fp32 scales that are stored."""
    n = np.asarray(data, dtype=np.float64)
    s = np.repeat(np.asarray(scale, dtype=np.float32).astype(np.float64), BLOCK, -1)
    return n * s[..., None]
