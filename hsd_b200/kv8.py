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

import ctypes as C
import math
from typing import NamedTuple

import torch

from . import _native as N
from .attention import _as_heads
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


_workspaces = {}
_FLAG_BYTES = 65536  # leading part of the workspace that starts as zeros


def _workspace(need, device):
    """Scratch of (device, current stream), grown to fit; its flags are zeroed
    once and every call leaves them ready for the next.  A call that is being
    captured into a graph gets scratch of its own, zeroed by the graph, so
    graphs that share no stream share no scratch either (replays of one graph
    never overlap)."""
    if torch.cuda.is_current_stream_capturing():
        buf = torch.empty(need + 256, dtype=torch.uint8, device=device)
        buf[:_FLAG_BYTES + 256].zero_()
        return buf
    key = (device.index, int(torch.cuda.current_stream(device).cuda_stream))
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < need + 256:
        buf = torch.zeros(max(need, 1 << 20) + 256, dtype=torch.uint8, device=device)
        _workspaces[key] = buf
    return buf


def _layer_tensors(layer, sealed, hkv, dev):
    """Addresses and strides of a layer's sealed rows, checked."""
    k8, v8, ks, vs = layer
    for t, name in ((k8, "k"), (v8, "v")):
        if t.dtype != torch.int8 or t.dim() != 3 or t.shape[0] != hkv or t.shape[2] != 128 \
                or t.shape[1] < sealed or t.stride(2) != 1 or t.stride(1) != 128:
            raise ValueError(f"layer.{name}: int8 [{hkv}, >= {sealed}, 128] with contiguous rows")
    for t, name in ((ks, "k_scale"), (vs, "v_scale")):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape[0] != hkv \
                or t.shape[1] < sealed // BLOCK or t.stride(1) != 1:
            raise ValueError(f"layer.{name}: float32 [{hkv}, >= {sealed // BLOCK}]")
    if hkv > 1 and ks.stride(0) != vs.stride(0):
        raise ValueError("layer: k_scale and v_scale must share a head stride")
    if any(t.device != dev for t in layer):
        raise ValueError(f"layer: tensors must be on {dev}")
    # the head stride of a single head is never used
    h8 = [t.stride(0) if hkv > 1 else t.shape[1] * 128 for t in (k8, v8)]
    return (N.ptr(k8), h8[0], N.ptr(v8), h8[1], N.ptr(ks), N.ptr(vs),
            ks.stride(0) if hkv > 1 else sealed // BLOCK)


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

    Runs on the device's current stream.  P is rounded to bf16 (as in
    :func:`verify_attention`); scores, sums and the joined partial rows are
    fp32.
    """
    q = _as_heads(q, "query")
    hq, q_len, d = q.shape
    dev, kv_len = q.device, plan.kv_len
    if d != 128:
        raise ValueError(f"query: head_dim {d} (128 only)")
    if not q.is_cuda or torch.device(plan.workspace.device) != dev:
        raise ValueError("query and plan must be on the same CUDA device")
    if plan.q_len != q_len:
        raise ValueError(f"plan is for {plan.q_len} rows, query has {q_len}")
    sealed, tail_row0 = int(sealed), int(tail_row0)
    if sealed < 0 or sealed % BLOCK or sealed > kv_len or not 0 <= tail_row0 <= sealed:
        raise ValueError(f"sealed={sealed} must be a multiple of {BLOCK} in [0, {kv_len}] and "
                         f"tail_row0={tail_row0} in [0, sealed]")
    if sealed < kv_len:
        if k is None or v is None:
            raise ValueError(f"columns {sealed}..{kv_len} need the bf16 tail")
        k, v = _as_heads(k, "key"), _as_heads(v, "value")
        hkv = k.shape[0]
        if v.shape[0] != hkv or k.shape[2] != 128 or v.shape[2] != 128 \
                or min(k.shape[1], v.shape[1]) < kv_len - tail_row0:
            raise ValueError(f"tail: key {tuple(k.shape)} and value {tuple(v.shape)} must be "
                             f"[Hkv, >= {kv_len - tail_row0}, 128]")
        if k.device != dev or v.device != dev:
            raise ValueError(f"tail: tensors must be on {dev}")
        # the head stride of a single head is never used
        tail = []
        for t in (k, v):
            tail += [N.ptr(t), t.stride(1), t.stride(0) if hkv > 1 else t.shape[1] * t.stride(1)]
    else:
        hkv = layer.k.shape[0]
        tail = [None, 0, 0, None, 0, 0]
    if hq % hkv:
        raise ValueError(f"{hq} query heads over {hkv} KV heads")
    if sealed:
        if layer is None:
            raise ValueError("sealed columns need the layer's tensors")
        sealed_args = _layer_tensors(layer, sealed, hkv, dev)
    else:
        sealed_args = (None, 0, None, 0, None, None, 0)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if out is None:
        out = torch.empty((q_len, hq, d), dtype=torch.bfloat16, device=dev)
    if need_lse and lse is None:
        lse = torch.empty((hq, q_len), dtype=torch.float32, device=dev)
    for t, dt, shape in ((out, torch.bfloat16, (q_len, hq, d)),
                         (lse if need_lse else None, torch.float32, (hq, q_len))):
        if t is not None and (t.dtype != dt or tuple(t.shape) != shape or not t.is_contiguous()
                              or t.device != dev):
            raise ValueError(f"output must be contiguous {dt} {shape} on {dev}")
    lib = N.load()
    with torch.cuda.device(dev):
        need = lib.hsd_kv8_attention_workspace_bytes(q_len, kv_len, hq, hkv)
        ws = _workspace(need, dev)
        N.check(lib.hsd_verify_attention_kv8(
            N.ptr(q), q.stride(1), q.stride(0) if hq > 1 else q_len * q.stride(1), *sealed_args[:7],
            sealed, *tail, tail_row0, N.ptr(out), N.ptr(lse) if need_lse else None, q_len, kv_len,
            hq, hkv, d, float(scale), C.byref(plan.struct),
            C.c_void_p((ws.data_ptr() + 255) & ~255), need, N.ptr(plan.status),
            N.stream_handle()), "hsd_verify_attention_kv8")
    return out, lse if need_lse else None
