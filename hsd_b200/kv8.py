"""A page's KV cache in 8 bits, with one scale for each 64-token block and head.

The verification loop reads the page prefix (image and prompt tokens) again
in every step of every layer, and never changes it: compaction moves rows at
or after the first dropped one, which lie behind the prefix.  So whole
64-token blocks of the prefix can be *sealed* -- stored as int8 with a scale
per block, plane (layer, K or V, KV head) -- while the rows behind them, the
*tail*, stay bf16 and are appended and compacted as before.  Should a compaction
reach sealed rows all the same, they have to leave the sealed ones
(:meth:`Kv8Cache.rows_moved`; ``loop.VerifyLoop(kv8=...)`` does it).  64
columns are the mask's tile width (BlockMask 128 x 64, D:94-106).

* :meth:`Kv8Cache.seal` / :meth:`Kv8Cache.unseal`: every layer in one launch;
* :func:`verify_attention_kv8`: the packed verification attention (the
  counterpart of :func:`hsd_b200.attention.verify_attention`) over sealed
  columns followed by the bf16 tail.

The reference has no such cache (its ``DynamicCache`` holds bf16, D:356-359).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N
from .plan import TilePlan

BLOCK = 64  # rows that share a scale


class Kv8Layer(NamedTuple):
    """One layer's sealed rows: int8 ``[Hkv, rows, 128]`` keys and values
    (contiguous rows) and their fp32 scales ``[Hkv, rows // 64]``."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor


class Kv8Cache:
    """The sealed rows of every layer.

    ``data``: int8 ``[layers, 2, Hkv, capacity, 128]``, ``scale``: fp32
    ``[layers, 2, Hkv, capacity // 64]``; the plane order is that of
    ``plane_pointers`` over the layers' K and V caches in turn.  ``sealed``
    rows (a multiple of 64) are in use, counted on the host when a call is made
    (or captured: a graph's replays seal the rows of the capture).  Calls run on
    the device's current stream; ``status`` (int32, one word per cache) collects
    device reports.
    """

    def __init__(self, layers, num_kv_heads, capacity, device="cuda"):
        if layers <= 0 or num_kv_heads <= 0 or capacity <= 0 or capacity % BLOCK:
            raise ValueError(f"Kv8Cache: {layers} layers, {num_kv_heads} heads, capacity "
                             f"{capacity} (a positive multiple of {BLOCK})")
        self.layers, self.num_kv_heads, self.capacity = layers, num_kv_heads, capacity
        self.data = torch.zeros(layers, 2, num_kv_heads, capacity, 128, dtype=torch.int8,
                                device=device)
        self.scale = torch.ones(layers, 2, num_kv_heads, capacity // BLOCK, dtype=torch.float32,
                                device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.sealed = 0

    def seal(self, planes, n_rows, src_row0=None):
        """Seal the next ``n_rows`` rows (a multiple of 64) of every plane,
        read from row ``src_row0`` on (default: the row of the same number).

        ``planes``: device addresses of the bf16 planes
        (``hsd_b200.compaction.plane_pointers`` over ``k0, v0, k1, v1, ...``).
        Infinities saturate and NaN become 0; either is reported
        (:meth:`raise_on_device_error`).
        """
        N.ops().kv8_seal(planes, self.sealed if src_row0 is None else src_row0, self.data,
                         self.scale, self.sealed, n_rows, self.status)
        self.sealed += n_rows

    def unseal(self, planes, row0, n_rows, dst_row0=None):
        """Rows ``[row0, row0 + n_rows)`` of every plane back as bf16, to rows
        ``dst_row0`` on (default: the same rows) of ``planes``; any row range
        of the sealed ones."""
        N.ops().kv8_unseal(self.data, self.scale, self.sealed, planes, row0, n_rows,
                           row0 if dst_row0 is None else dst_row0)

    def reset(self, sealed=0):
        """Keep only the first ``sealed`` rows (a multiple of 64)."""
        if sealed < 0 or sealed % BLOCK or sealed > self.sealed:
            raise ValueError(f"reset: {sealed} of {self.sealed} sealed rows")
        self.sealed = sealed

    def rows_moved(self, first):
        """The planes' rows from ``first`` on have been moved or dropped (a
        compaction; ``counts[1]`` of :func:`hsd_b200.compaction.keep_indices`):
        keep the blocks in front of it.  Returns the rows still sealed."""
        if first < 0:
            raise ValueError(f"rows_moved: row {first}")
        self.sealed = min(self.sealed, first // BLOCK * BLOCK)
        return self.sealed

    def layer(self, l) -> Kv8Layer:
        """Layer ``l``'s tensors (views), for :func:`verify_attention_kv8`."""
        d, s = self.data[l], self.scale[l]
        return Kv8Layer(d[0], d[1], s[0], s[1])

    def raise_on_device_error(self):
        """Raise, and clear the report, if a call since the last one sealed an
        infinity or NaN."""
        code = int(self.status.item())
        if code:
            self.status.zero_()
            raise N.HSDError(f"device status 0x{code:x} while sealing (0x{N.HSD_DEV_BAD_VALUE:x}: "
                             "an infinity or NaN among the rows)")


def verify_attention_kv8(q, layer, sealed, k, v, plan: TilePlan, scale=None, tail_row0=0,
                         out=None, lse=None, need_lse=True):
    """Masked GQA attention over a tile plan whose first ``sealed`` columns
    are held in 8 bits, the counterpart of
    :func:`hsd_b200.attention.verify_attention`.

    q: ``[Hq, Q, 128]`` (or ``[1, Hq, Q, 128]``) bf16, any row / head strides;
    layer: the :class:`Kv8Layer` of the sealed columns (None when ``sealed``
    is 0); k, v: ``[Hkv, rows, 128]`` bf16, column ``c >= sealed`` being row
    ``c - tail_row0`` (``tail_row0=0``: full caches, whose sealed rows are not
    read; ``tail_row0=sealed``: the rows behind them alone; None when every
    column is sealed).  ``scale`` (default ``128 ** -0.5``) must be positive.
    Returns ``(out [Q, Hq, 128] bf16, lse [Hq, Q] fp32 natural log or None)``;
    rows that see nothing give 0 and -inf.

    Runs on the device's current stream, with 2 MB of scratch kept per device
    and stream; with many rows the layer's expanded columns (512 bytes per
    column and KV head) are held for the call, from PyTorch's allocator.  Scales must not be negative; 0 stands for a
    block of zeros.  P is rounded to fp16 (few rows: to bf16 over the bf16
    columns); scores and sums are fp32.  V's blocks of 64 columns may differ by
    2^60 in magnitude, from 2^-73 to 2^80 (beside blocks of zeros: to 2^48).
    """
    return N.ops().verify_attention_kv8(q, layer, sealed, k, v, plan.address, plan.status, scale,
                                        tail_row0, out, lse, need_lse)
