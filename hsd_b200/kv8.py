"""A page's KV cache in 8 bits, with one scale for each 64-token block and head.

The verification loop reads the page prefix (image and prompt tokens) again
in every step of every layer, and never changes it: compaction moves rows at
or after the first dropped one, which lie behind the prefix.  So whole
64-token blocks of the prefix can be *sealed* -- stored as int8 with a scale
per block, plane (layer, K or V, KV head) -- while the rows behind them, the
*tail*, stay bf16 and are appended and compacted as before.  64 columns are
the mask's tile width (BlockMask 128 x 64, D:94-106).

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
    rows (a multiple of 64) are in use.  Calls run on the device's current
    stream; ``status`` (int32, one word per cache) collects device reports.
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

    def _planes(self, planes, what):
        n = self.layers * 2 * self.num_kv_heads
        if planes.dtype != torch.int64 or planes.numel() != n or not planes.is_contiguous():
            raise ValueError(f"{what}: {n} plane addresses (int64) are needed")
        if planes.device != self.data.device:
            raise ValueError(f"{what}: the planes' addresses must be on {self.data.device}")

    def seal(self, planes, n_rows, src_row0=None):
        """Seal the next ``n_rows`` rows (a multiple of 64) of every plane,
        read from row ``src_row0`` on (default: the row of the same number).

        ``planes``: device addresses of the bf16 planes
        (``hsd_b200.compaction.plane_pointers`` over ``k0, v0, k1, v1, ...``).
        Infinities saturate and NaN become 0; either is reported
        (:meth:`raise_on_device_error`).
        """
        self._planes(planes, "seal")
        row0 = self.sealed if src_row0 is None else int(src_row0)
        if n_rows < 0 or n_rows % BLOCK or self.sealed + n_rows > self.capacity or row0 < 0:
            raise ValueError(f"seal: {n_rows} rows from {row0} (a multiple of {BLOCK}) after "
                             f"{self.sealed} of {self.capacity}")
        with torch.cuda.device(self.data.device):
            N.check(N.load().hsd_kv8_seal(
                N.ptr(planes), planes.numel(), row0, N.ptr(self.data), self.data.stride(2),
                N.ptr(self.scale), self.scale.stride(2), self.sealed // BLOCK, n_rows // BLOCK,
                N.ptr(self.status), N.stream_handle()), "hsd_kv8_seal")
        self.sealed += n_rows

    def unseal(self, planes, row0, n_rows, dst_row0=None):
        """Rows ``[row0, row0 + n_rows)`` of every plane back as bf16, to rows
        ``dst_row0`` on (default: the same rows) of ``planes``; any row range
        of the sealed ones."""
        self._planes(planes, "unseal")
        dst = row0 if dst_row0 is None else int(dst_row0)
        if row0 < 0 or n_rows < 0 or row0 + n_rows > self.sealed or dst < 0:
            raise ValueError(f"unseal: rows {row0}..{row0 + n_rows} of {self.sealed} to {dst}")
        with torch.cuda.device(self.data.device):
            N.check(N.load().hsd_kv8_unseal(
                N.ptr(self.data), self.data.stride(2), N.ptr(self.scale), self.scale.stride(2),
                planes.numel(), row0, n_rows, N.ptr(planes), dst, N.stream_handle()),
                "hsd_kv8_unseal")

    def reset(self, sealed=0):
        """Keep only the first ``sealed`` rows (a multiple of 64)."""
        if sealed < 0 or sealed % BLOCK or sealed > self.sealed:
            raise ValueError(f"reset: {sealed} of {self.sealed} sealed rows")
        self.sealed = sealed

    def layer(self, l) -> Kv8Layer:
        """Layer ``l``'s tensors (views), for :func:`verify_attention_kv8`."""
        d, s = self.data[l], self.scale[l]
        return Kv8Layer(d[0], d[1], s[0], s[1])

    def raise_on_device_error(self):
        code = int(self.status.item())
        if code:
            raise N.HSDError(f"device status 0x{code:x} while sealing (0x{N.HSD_DEV_BAD_VALUE:x}: "
                             "an infinity or NaN among the rows)")
