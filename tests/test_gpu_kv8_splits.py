"""Every way in which the few-rows kernel of the 8-bit attention divides a tile's
columns: clusters of each size from 1 to 16 with steps of 32 columns, of each size
that takes steps of 64, and the second launch; with 8 and 16 packed rows a tile.
The choice made is asserted, so that another time model cannot silently leave
one out.

Oracle and limits: ``tests/test_gpu_kv8_attention.py``.
"""
import ctypes as C

import pytest
import torch

from tests import test_gpu_kv8_attention as T

pytestmark = pytest.mark.gpu
dev = T.dev

# q_len, heads: 8 and 16 packed rows a tile
NARROW, WIDE = (1, 1, 1), (2, 5, 1)
CASES = [(*r, 256 * s - 90, s, False, 32) for r in (NARROW, WIDE) for s in range(1, 17)]
CASES += [(*r, 512 * s - 90, s, False, 64) for r in (NARROW, WIDE) for s in range(9, 17)]
CASES += [(q, 16, 8, 512 * s - 90, s, False, 64) for q in (1, 5) for s in (6, 7, 8)]
CASES += [(5, 28, 4, 2470, 5, False, 64), (10, 16, 8, 1958, 4, False, 64),
          (20, 16, 8, 1446, 3, False, 64), (64, 12, 2, 934, 2, False, 64),
          (100, 12, 2, 422, 1, False, 64)]
CASES += [(*NARROW, 8300, 33, True, 32), (1, 4, 4, 9600, 19, True, 64), (*WIDE, 8300, 33, True, 32),
          (3, 6, 2, 19000, 38, True, 64)]


def choice(q_len, kv_len, hq, hkv):
    from hsd_b200 import _native as N
    c = (C.c_int32 * 4)()
    N.check(N.load().hsd_kv8_attention_choice(q_len, kv_len, hq, hkv, c), "choice")
    return tuple(c)


@pytest.mark.parametrize("q_len,hq,hkv,kv_len,ctas,join,step", CASES)
def test_split(dev, q_len, hq, hkv, kv_len, ctas, join, step):
    assert choice(q_len, kv_len, hq, hkv) == (0, ctas, join, step)
    sealed = (kv_len - q_len - 20) // 64 * 64
    allowed = T.segments([q_len], kv_len - q_len)
    g = torch.Generator().manual_seed(kv_len)
    allowed &= torch.rand(allowed.shape, generator=g) < 0.9
    allowed[0, 64:kv_len // 2] = False       # CTAs without a column of row 0
    x = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=kv_len)
    allowed = allowed.to(dev)
    T.check(T.run(*x, sealed, T.plan_of(allowed)), T.exact(*x, sealed, allowed))


def test_choice_of_many_rows_and_refusals(dev):
    from hsd_b200 import _native as N
    assert choice(2176, 4800, 12, 2) == (1, 0, 0, 0)
    c = (C.c_int32 * 4)()
    lib = N.load()
    for bad in ((0, 300, 12, 2), (64, 0, 12, 2), (64, 300, 12, 5), (64, 300, 12, 0)):
        assert lib.hsd_kv8_attention_choice(*bad, c) == 1
    assert lib.hsd_kv8_attention_choice(64, 300, 12, 2, None) == 1
