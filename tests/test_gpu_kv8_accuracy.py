"""How near the 8-bit attention comes where its P is fp16: sealed columns (few
rows), sealed and bf16 ones (many rows).

Limits, from the arithmetic.  Rounding the output to bf16 is off by r0, which
the oracle gives exactly.  P's rounding to fp16 is off by at most 2^-11 of each
weight, evenly spread and independent: 2^-11 / sqrt(3) sqrt(sum w^2 v^2) rms.  A
score's fp32 errors reach the weights as 2^-18 (largest |score| + 1) of them.
Many rows: the partial rows of items cut between CTAs are fp16 times a power of
two per row, 2^-11 of the row's largest value at most, their shares adding up to
1.  Independent errors add in squares; 5 % for the sampling of r0.  (P in bf16
would be off by 2^-8 / sqrt(3) sqrt(sum w^2 v^2), about as much as r0.)
"""
import math

import pytest
import torch

from tests import test_gpu_kv8_attention as T
from tests.test_gpu_kv8_attention_many import many

pytestmark = pytest.mark.gpu
dev = T.dev


@pytest.mark.parametrize("q_len,kv_len,sealed,hq,hkv,is_many", [
    (1, 2624, 2624, 12, 2, False), (1, 20032, 20032, 16, 8, False), (40, 2624, 2624, 12, 2, False),
    (9, 6400, 6400, 5, 1, False), (900, 2000, 1984, 12, 2, True), (700, 4000, 1024, 5, 1, True),
    (2049, 6000, 5952, 12, 2, True), (300, 16384, 16384, 8, 1, True),
    (1000, 1500, 0, 16, 8, True),
])
def test_near_the_outputs_own_rounding(dev, q_len, kv_len, sealed, hq, hkv, is_many):
    assert many(q_len, kv_len, hq, hkv) == is_many
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=kv_len)
    allowed = (torch.rand(q_len, kv_len, generator=torch.Generator().manual_seed(1)) < 0.8).to(dev)
    got, _ = T.run(q, data, scale, tail, sealed, T.plan_of(allowed))
    kv = torch.cat([data[:, :, :sealed].double()
                    * scale[..., :sealed // 64].double().repeat_interleave(64, -1)[..., None],
                    tail[:, :, sealed:kv_len].double()], 2)
    err2 = r02 = p2 = s2 = rec2 = 0.0
    for h in range(hq):
        k, v = kv[0, h * hkv // hq], kv[1, h * hkv // hq]
        s = (q[h].double() @ k.t()) / math.sqrt(128)
        top = float(s.abs().max())
        w = torch.softmax(s.masked_fill(~allowed, -math.inf), -1)
        want = w @ v
        err2 += float((got[:, h].double() - want).pow(2).sum())
        r02 += float((want.to(torch.bfloat16).double() - want).pow(2).sum())
        p2 += float((w.pow(2) @ v.pow(2)).sum()) * 2.0 ** -22 / 3
        s2 += float((w @ v.abs()).pow(2).sum()) * (2.0 ** -18 * (top + 1)) ** 2
        if is_many:
            rec2 += 128 * float(want.abs().amax(-1).pow(2).sum()) * 2.0 ** -22
    limit = 1.05 ** 2 * r02 + p2 + s2 + rec2
    print(f"error {math.sqrt(err2 / limit):.3f} of the limit, {math.sqrt(err2 / r02):.3f} r0")
    assert err2 <= limit
