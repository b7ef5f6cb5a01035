"""Verification attention with odd head groups and several pieces per CTA.

A KV group of 3, 5 or 7 query heads gives one item per group with a single
head; a CTA whose work holds such an item between items of two heads has one
slot idle for it, and the idle slot's tiles must still pass it in step.
Against 64 bits; the tolerance is that of bf16 P (2^-7 of the largest visible
value) and of the output's rounding.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from hsd_b200 import _native
    _native.load()
    return torch.device("cuda:0")


@pytest.mark.parametrize("hq,hkv,q_len,kv_len", [
    (7, 1, 3000, 3400), (28, 4, 1025, 1088), (15, 3, 2000, 2100), (9, 3, 4000, 4096),
])
def test_odd_groups(dev, hq, hkv, q_len, kv_len):
    from hsd_b200.attention import verify_attention
    from hsd_b200.plan import SEG_CAUSAL, PackedMask
    import numpy as np
    g = torch.Generator(device=dev).manual_seed(hq)
    q = torch.randn(hq, q_len, 128, generator=g, device=dev).to(torch.bfloat16)
    k = torch.randn(hkv, kv_len, 128, generator=g, device=dev).to(torch.bfloat16)
    v = torch.randn(hkv, kv_len, 128, generator=g, device=dev).to(torch.bfloat16)
    prefix = kv_len - q_len
    plan = PackedMask(q_len, kv_len, [dict(q_start=0, q_len=q_len, kind=SEG_CAUSAL,
                                           kv=np.arange(kv_len) < prefix)], device=dev).plan()
    out, lse = verify_attention(q, k, v, plan)
    torch.cuda.synchronize()
    plan.raise_on_device_error()
    i = torch.arange(q_len, device=dev)[:, None] + prefix
    hide = torch.arange(kv_len, device=dev)[None] > i
    for h in range(hq):
        s = (q[h].double() @ k[h * hkv // hq].double().t()) / math.sqrt(128)
        s = s.masked_fill(hide, -math.inf)
        vv = v[h * hkv // hq].double()
        want = torch.softmax(s, -1) @ vv
        err = (out[:, h].double() - want).abs()
        assert float((err - 2.0 ** -7 * vv.abs().max() - 2.0 ** -7 * want.abs()).max()) <= 0
        assert err.pow(2).mean().sqrt() <= 3 * 2.0 ** -8 * want.pow(2).mean().sqrt()
        w = torch.logsumexp(s, -1)
        assert float((lse[h].double() - w).abs().max()) <= 2.0 ** -18 * (
            float(s[~hide].abs().max()) + float(w.abs().max()) + 1)
