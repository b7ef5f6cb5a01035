"""A model that normalises queries and keys per head after the rotation: the norm
is the caller's, on the returned view and on the rows just written."""
import math

import numpy as np
import pytest
import torch

from oracle import rope_axes as OA

pytestmark = pytest.mark.gpu


def test_norm_between_rotation_and_attention():
    """Tolerance: the rotated value's bf16 rounding and the normalised one's, 2^-8 each
    of the largest of a head (the norm's factor moves with all 128 of them)."""
    from hsd_b200.attention import verify_attention
    from hsd_b200.plan import SEG_CAUSAL, PackedMask
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    dev = torch.device("cuda:0")
    hq, hkv, n, at, sections = 4, 2, 70, 30, [16, 16, 16, 16]
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(n, (hq + 2 * hkv) * 128, generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 5000, (1, 4, n), generator=g)
    w = torch.rand(2, 128, generator=g) + 0.5
    kc = torch.randn(hkv, at + n + 3, 128, generator=g).to(torch.bfloat16).to(dev)
    vc = torch.randn(hkv, at + n + 3, 128, generator=g).to(torch.bfloat16).to(dev)
    kc0 = kc.clone()
    q_norm, k_norm = (torch.nn.RMSNorm(128, eps=1e-5, device=dev, dtype=torch.float32)
                      for _ in range(2))
    q_norm.weight.data.copy_(w[0])
    k_norm.weight.data.copy_(w[1])
    x = qkv.to(dev)
    a, b = hq * 128, (hq + hkv) * 128
    q = rope_append_axes(x[:, :a], x[:, a:b], x[:, b:], pos.to(dev),
                         RotaryAxes(sections, device=dev), kc, vc, at)
    with torch.no_grad():
        q = q_norm(q.float()).to(torch.bfloat16)
        new = kc[:, at:at + n]
        new.copy_(k_norm(new.float()))
    freq = [1e6 ** (-i / 64) for i in range(64)]
    rot = OA.rotate(qkv[:, :b].double().numpy().reshape(n, hq + hkv, 128), pos[0].numpy(),
                    OA.pair_axis(sections), freq)
    rms = np.sqrt((rot ** 2).mean(-1, keepdims=True) + 1e-5)
    rot = rot / rms * np.concatenate([np.repeat(w[:1].numpy(), hq, 0), np.repeat(w[1:].numpy(), hkv, 0)])[None]
    got = np.concatenate([q[0].transpose(0, 1).double().cpu().numpy(),
                          kc[:, at:at + n].transpose(0, 1).double().cpu().numpy()], 1)
    assert (np.abs(got - rot) <= 2.0 ** -7 * np.abs(rot).max(-1, keepdims=True)).all()
    assert torch.equal(kc[:, :at], kc0[:, :at]) and torch.equal(kc[:, at + n:], kc0[:, at + n:])
    # the normalised queries and rows are what the attention takes
    seen = np.arange(at + n) < at
    plan = PackedMask(n, at + n, [dict(q_start=0, q_len=n, kind=SEG_CAUSAL, kv=seen)],
                      device=dev).plan()
    out, _ = verify_attention(q, kc[:, :at + n], vc[:, :at + n], plan)
    hide = torch.arange(at + n, device=dev)[None] > torch.arange(n, device=dev)[:, None] + at
    for h in range(hq):
        k, v = kc[h * hkv // hq, :at + n].double(), vc[h * hkv // hq, :at + n].double()
        s = (q[0, h].double() @ k.t() / math.sqrt(128)).masked_fill(hide, -math.inf)
        want = torch.softmax(s, -1) @ v
        assert ((out[:, h].double() - want).abs()
                <= 2.0 ** -7 * (v.abs().max() + want.abs())).all()
