"""Scratch of the 8-bit attention: what a call holds is PyTorch's again after it."""
import pytest
import torch

from tests import test_gpu_kv8_attention as T
from tests.test_gpu_kv8_attention_many import many

pytestmark = pytest.mark.gpu
dev = T.dev


def test_many_rows_leave_no_scratch_behind(dev):
    """A layer's expanded columns (and partial records) do not stay allocated, on
    any stream; calls that follow one another at once keep their results."""
    hq, hkv, q_len, kv_len, sealed = 8, 8, 700, 20000, 19968
    assert many(q_len, kv_len, hq, hkv)
    allowed = T.segments([q_len], kv_len - q_len).to(dev)
    x = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=3)
    plan = T.plan_of(allowed)
    want = T.run(*x, sealed, plan)
    T.check(want, T.exact(*x, sealed, allowed))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(dev)
    for s in streams:
        with torch.cuda.stream(s):
            got = [T.run(*x, sealed, plan) for _ in range(2)]
            fill = torch.full((512 * hkv * kv_len,), 255, dtype=torch.uint8, device=dev)
            s.synchronize()
        for o, l in got:
            assert torch.equal(o, want[0]) and torch.equal(l, want[1])
        del got, fill, o, l
    assert torch.cuda.memory_allocated(dev) - before <= len(streams) * (3 << 20)
    # back to back without a wait, the allocator's block reused by what follows
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    layer = Kv8Layer(x[1][0], x[1][1], x[2][0], x[2][1])
    outs = []
    for _ in range(4):
        outs.append(verify_attention_kv8(x[0], layer, sealed, x[3][0], x[3][1], plan))
        torch.full((512 * hkv * kv_len,), 255, dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    for o, l in outs:
        assert torch.equal(o, want[0]) and torch.equal(l, want[1])


def test_few_rows_fit_the_kept_scratch(dev):
    """Whatever the sizes, a few-rows call needs at most the 2 MB that are kept."""
    from hsd_b200 import _native as N
    lib = N.load()
    for hq, hkv in ((12, 2), (16, 8), (8, 1), (4, 4), (28, 4), (5, 1), (32, 8), (64, 64)):
        for q_len in (1, 2, 5, 17, 40, 100):
            for kv_len in (65, 1000, 8193, 40000, 131072, 1 << 20):
                need = lib.hsd_kv8_attention_workspace_bytes(q_len, kv_len, hq, hkv)
                assert need <= 2 << 20 or need >= 512 * hkv * kv_len


def test_out_of_memory_is_pytorchs_error(dev):
    """With PyTorch's own limit set (nothing is allocated beyond it), a call that
    cannot have its scratch raises torch.OutOfMemoryError, and runs once it can."""
    hq, hkv, q_len, kv_len, sealed = 8, 8, 700, 20000, 19968
    assert many(q_len, kv_len, hq, hkv)
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    x = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=3)
    plan = T.plan_of(allowed)
    want = T.run(*x, sealed, plan)
    torch.cuda.synchronize()
    del allowed
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(dev).total_memory
    try:
        torch.cuda.set_per_process_memory_fraction(
            (torch.cuda.memory_reserved(dev) + (24 << 20)) / total, dev)
        held = []                         # what the allocator still has free
        for size in (32 << 20, 4 << 20):
            with pytest.raises(torch.OutOfMemoryError):
                for _ in range(1000):
                    held.append(torch.empty(size, dtype=torch.uint8, device=dev))
        with pytest.raises(torch.OutOfMemoryError):
            T.run(*x, sealed, plan)
        del held
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0, dev)
    got = T.run(*x, sealed, plan)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
