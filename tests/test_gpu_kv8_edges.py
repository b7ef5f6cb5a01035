"""The 8-bit attention where factors vanish: zero query rows, blocks and scales
of zero, V of unlike size beside blocks of zeros.

Oracle and limits: ``tests/test_gpu_kv8_attention.py``.
"""
import pytest
import torch

from tests import test_gpu_kv8_attention as T
from tests.test_gpu_kv8_attention_many import many

pytestmark = pytest.mark.gpu
dev = T.dev

# few rows (8 and 16 a tile) and many
ROWS = [(1, 4, 2, False), (11, 5, 1, False), (30, 12, 2, False), (900, 12, 2, True)]


@pytest.mark.parametrize("q_len,hq,hkv,is_many", ROWS)
@pytest.mark.parametrize("sm", [None, 1e-20])
def test_zero_query_rows_over_zero_keys(dev, q_len, hq, hkv, is_many, sm):
    """A zero query row (unit 2^-100) against a block of zero keys (scale
    2^-100 / 127) or under a tiny softmax scale: the score factor is below fp32's
    range, and masked columns still have to vanish."""
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    kv_len, sealed = 500, 448
    assert many(q_len, kv_len, hq, hkv) == is_many
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=q_len)
    q[:, ::2] = 0
    for b in (1, 2, 5):
        data[0, :, 64 * b:64 * b + 64] = 0
        scale[0, :, b] = 2.0 ** -100 / 127
    g = torch.Generator().manual_seed(1)
    allowed = (torch.rand(q_len, kv_len, generator=g) < 0.5).to(dev)
    allowed[0, 64:192] = False            # nothing of two of the blocks
    allowed[1::3] = False                 # rows that see nothing ...
    allowed[3::6, 70:75] = True           # ... or a few zero keys alone
    plan = T.plan_of(allowed)
    got = verify_attention_kv8(q, Kv8Layer(data[0], data[1], scale[0], scale[1]), sealed, tail[0],
                               tail[1], plan, scale=sm)
    torch.cuda.synchronize()
    plan.raise_on_device_error()
    T.check(got, T.exact(q, data, scale, tail, sealed, allowed, sm=sm))


@pytest.mark.parametrize("q_len,hq,hkv,is_many", ROWS)
def test_bf16_block_of_zeros_beside_small_values(dev, q_len, hq, hkv, is_many):
    """V of 2^-30 with a visible block of zeros among the bf16 columns: the zeros
    take part in the weights and cost the others none of their bits."""
    kv_len, sealed = 640, 320
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=q_len)
    scale[1] *= 2.0 ** -30
    tail[1] *= 2.0 ** -30
    tail[1, :, 384:448] = 0
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    got = T.run(q, data, scale, tail, sealed, T.plan_of(allowed))
    T.check(got, T.exact(q, data, scale, tail, sealed, allowed))


@pytest.mark.parametrize("q_len", [1, 3])
@pytest.mark.parametrize("big", [20, 60, 90])
def test_sealed_zeros_beside_large_values_few_rows(dev, q_len, big):
    """Blocks of zeros (scale 2^-100 / 127) beside V of 2^big, several of each to a
    warp: their quotient is past fp32's range, their weights still count."""
    hq, hkv, kv_len, sealed = 16, 8, 20000, 19968
    assert not many(q_len, kv_len, hq, hkv)
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=q_len)
    scale[1] *= 2.0 ** big
    tail[1] = (tail[1].float() * 2.0 ** big).to(torch.bfloat16)
    g = torch.Generator().manual_seed(big)
    zero = (torch.rand(sealed // 64, generator=g) < 0.5).to(dev)
    data[1, :, :sealed][:, zero.repeat_interleave(64)] = 0
    scale[1, :, :sealed // 64][:, zero] = 2.0 ** -100 / 127
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    allowed[-1, 64:192] = False
    T.check(T.run(q, data, scale, tail, sealed, T.plan_of(allowed)),
            T.exact(q, data, scale, tail, sealed, allowed))


@pytest.mark.parametrize("q_len,hq,hkv,is_many", ROWS)
@pytest.mark.parametrize("everywhere", [False, True])
def test_scales_of_zero(dev, q_len, hq, hkv, is_many, everywhere):
    """Another quantiser's scale of a block of zeros: the block's keys and values
    are zeros, whatever its bytes."""
    kv_len, sealed = 500, 448
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=q_len)
    g = torch.Generator().manual_seed(2)
    allowed = (torch.rand(q_len, kv_len, generator=g) < 0.6).to(dev)
    allowed[0] = False
    allowed[0, :100] = True
    if everywhere:
        scale[:] = 0
        allowed[:, sealed:] = False
    else:
        scale[0, :, [0, 2, 6]] = 0
        scale[1, :, [0, 1, 5]] = 0
    got = T.run(q, data, scale, tail, sealed, T.plan_of(allowed))
    T.check(got, T.exact(q, data, scale, tail, sealed, allowed))
    if everywhere:
        assert bool((got[0] == 0).all())


@pytest.mark.parametrize("tail_zeros", [False, True])
def test_zeros_beside_large_values_many_rows(dev, tail_zeros):
    """Zeros beside V of 2^25 at most, sealed and bf16: their weights still count,
    down to 2^-24 of a row's largest."""
    q_len, hq, hkv, kv_len, sealed = 900, 12, 2, 1000, 640
    assert many(q_len, kv_len, hq, hkv)
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=1)
    scale[1] *= 2.0 ** 22
    tail[1] = (tail[1].float() * 2.0 ** 22).to(torch.bfloat16)
    for b in (0, 3, 4, 8):
        data[1, :, 64 * b:64 * b + 64] = 0
        scale[1, :, b] = 2.0 ** -100 / 127
    if tail_zeros:
        tail[1, :, 704:832] = 0
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    allowed[-1, 64:192] = False
    T.check(T.run(q, data, scale, tail, sealed, T.plan_of(allowed)),
            T.exact(q, data, scale, tail, sealed, allowed))


@pytest.mark.parametrize("q_len,hq,hkv", [(634, 7, 1), (900, 12, 2)])
@pytest.mark.parametrize("big", [14, 40])
def test_zeros_keep_their_weights_when_items_are_joined(dev, q_len, hq, hkv, big):
    """A sealed prefix of zeros (scores of 0) and bf16 columns with V of 2^big and
    scores up to 20: the prefix's share of the sum, e^-15 a column, outlives the
    join of an item's parts, some of which hold nothing but zeros."""
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    kv_len, sealed = 9013, 2496
    assert many(q_len, kv_len, hq, hkv)
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=big)
    data[:] = 0
    scale[:] = 2.0 ** -100 / 127
    tail[1] = (tail[1].float() * 2.0 ** big).to(torch.bfloat16)
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    plan = T.plan_of(allowed)
    got = verify_attention_kv8(q, Kv8Layer(data[0], data[1], scale[0], scale[1]), sealed, tail[0],
                               tail[1], plan, scale=0.3)
    torch.cuda.synchronize()
    plan.raise_on_device_error()
    T.check(got, T.exact(q, data, scale, tail, sealed, allowed, sm=0.3))


@pytest.mark.parametrize("small", [-40, -60])
def test_small_values_many_rows(dev, small):
    """V of 2^small throughout, sealed and bf16: the least factor on V costs it nothing."""
    q_len, hq, hkv, kv_len, sealed = 900, 12, 2, 1000, 640
    assert many(q_len, kv_len, hq, hkv)
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=1)
    scale[1] *= 2.0 ** small
    tail[1] = (tail[1].float() * 2.0 ** small).to(torch.bfloat16)
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    T.check(T.run(q, data, scale, tail, sealed, T.plan_of(allowed)),
            T.exact(q, data, scale, tail, sealed, allowed))
