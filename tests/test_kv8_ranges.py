"""Row ranges of the 8-bit cache and the rotary update that pass 64 bits: refused
on the host, where their ends would wrap around to small numbers.  No GPU needed."""
import ctypes as C

import pytest
import torch

from hsd_b200 import _native as N

A = C.c_void_p(256)
FAR = 2 ** 63 - 1


def test_kv8_ranges_that_wrap_are_refused():
    lib = N.load()

    def seal(n=1, row0=0, block0=0, blocks=1, stride=64 * 128):
        return lib.hsd_kv8_seal(A, n, row0, A, stride, A, 1, block0, blocks, None, None)

    def unseal(n=1, row0=0, rows=64, dst=0, stride=64 * 128):
        return lib.hsd_kv8_unseal(A, stride, A, 1, n, row0, rows, A, dst, None)

    for n in (1, 4):
        for rc in (seal(n, row0=FAR), seal(n, row0=2 ** 56), unseal(n, row0=FAR),
                   unseal(n, row0=FAR - 63), unseal(n, row0=2 ** 56), unseal(n, dst=FAR),
                   unseal(n, dst=2 ** 55)):
            assert rc == 1, (n, rc, lib.hsd_last_error())
            assert b"range" in lib.hsd_last_error()


def test_kv8_cache_ranges_that_wrap_are_refused():
    from hsd_b200.kv8 import Kv8Cache
    c = Kv8Cache(2, 2, 256, device="cpu")
    planes = torch.zeros(8, dtype=torch.int64)
    c.sealed = 128
    for row0, n in ((FAR, 64), (FAR - 10, 64), (64, FAR), (1, FAR)):
        with pytest.raises(ValueError):
            c.unseal(planes, row0, n, dst_row0=0)
    for n in (2 ** 63 - 64, 2 ** 62):
        with pytest.raises(ValueError):
            c.seal(planes, n)
    for row0 in (FAR, 2 ** 56):
        with pytest.raises(ValueError):
            c.seal(planes, 64, src_row0=row0)
        with pytest.raises(ValueError):
            c.unseal(planes, 0, 64, dst_row0=row0)
    assert c.sealed == 128


def test_rope_axes_rows_that_wrap_are_refused():
    lib = N.load()
    for row0 in (FAR, 2 ** 56):
        assert lib.hsd_rope_append_axes(A, 1536, A, 1536, A, 256, A, 256, A, 4, 1, 3, A, A, 1.0, 4, 12,
                                        2, 128, A, 4096, A, 4096, 128, row0, None, None) == 1
        assert b"bad arguments" in lib.hsd_last_error()


@pytest.mark.gpu
def test_rope_axes_rows_past_the_cache_are_refused():
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    dev = torch.device("cuda:0")
    rot = RotaryAxes([64], device=dev)
    x = torch.ones(4, 256, dtype=torch.bfloat16, device=dev)
    kc = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    pos = torch.zeros(1, 4, dtype=torch.int64, device=dev)
    for row0 in (FAR, FAR - 3, 2 ** 62, 5, -1, -FAR):
        with pytest.raises(ValueError):
            rope_append_axes(x, x, x, pos, rot, kc, vc, row0)
    rope_append_axes(None, x, x, pos, rot, kc, vc, 4)
    assert bool((kc[:, 4:] == 1).all()) and not kc[:, :4].any()


@pytest.mark.gpu
def test_rope_axes_caches_with_heads_in_one_place_are_refused():
    """Expanded caches: every head would be written to the same rows."""
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    dev = torch.device("cuda:0")
    rot = RotaryAxes([64], device=dev)
    x = torch.ones(4, 256, dtype=torch.bfloat16, device=dev)
    kc = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device=dev)
    pos = torch.zeros(1, 4, dtype=torch.int64, device=dev)
    one_head = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=dev).expand(2, 8, 128)
    one_row = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device=dev).expand(2, 8, 128)
    for k_cache, v_cache in ((one_head, kc), (kc, one_head), (one_row, one_row)):
        with pytest.raises((ValueError, N.HSDError)):
            rope_append_axes(None, x, x, pos, rot, k_cache, v_cache, 0)
    torch.cuda.synchronize()
    assert not kc.any() and not one_head.any() and not one_row.any()
