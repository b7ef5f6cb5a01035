"""A cache used for page after page: one page's report does not stay for the next."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_report_is_raised_once():
    from hsd_b200 import _native as N
    from hsd_b200.compaction import plane_pointers
    from hsd_b200.kv8 import Kv8Cache
    dev = torch.device("cuda:0")
    x = torch.randn(2, 1, 128, 128, device=dev).to(torch.bfloat16)
    bad = x.clone()
    bad[1, 0, 100, 3] = float("nan")
    kv8 = Kv8Cache(1, 1, 128, device=dev)
    kv8.seal(plane_pointers([bad[0], bad[1]]), 64)
    kv8.raise_on_device_error()                       # the first block is clean
    kv8.seal(plane_pointers([bad[0], bad[1]]), 64)
    with pytest.raises(N.HSDError, match="infinity"):
        kv8.raise_on_device_error()
    kv8.reset()
    kv8.seal(plane_pointers([x[0], x[1]]), 128)
    kv8.raise_on_device_error()
    kv8.reset(64)
    kv8.seal(plane_pointers([bad[0], bad[1]]), 64)
    with pytest.raises(N.HSDError, match="infinity"):
        kv8.raise_on_device_error()
