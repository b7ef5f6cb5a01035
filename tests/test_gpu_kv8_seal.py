"""GPU parity of the 8-bit cache's sealing and unsealing: integers and scales
equal to the 64-bit oracle's, unsealed rows to the rounded products."""
import numpy as np
import pytest
import torch

from oracle import kv8 as OK

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from hsd_b200 import _native
    _native.load()
    return torch.device("cuda:0")


def _cache(dev, caches, capacity):
    from hsd_b200.compaction import plane_pointers
    from hsd_b200.kv8 import Kv8Cache
    kv8 = Kv8Cache(len(caches) // 2, caches[0].shape[-3], capacity, device=dev)
    return kv8, plane_pointers(caches)


def _check(kv8, x, lo, hi):
    """x: [L, 2, Hkv, rows, 128] bf16, sealed as rows [lo, hi)"""
    n, s = OK.seal(x.cpu())
    got = kv8.data[:, :, :, lo:hi].cpu().numpy()
    assert np.array_equal(got, n)
    assert np.array_equal(kv8.scale[..., lo // 64:hi // 64].cpu().numpy(), s.astype(np.float32))


@pytest.mark.parametrize("layers,hkv,rows,capacity,seed", [
    (1, 1, 64, 64, 0), (3, 2, 320, 448, 1), (28, 2, 128, 128, 2), (2, 8, 64, 1024, 3),
])
def test_seal_matches_oracle_and_unseal(dev, layers, hkv, rows, capacity, seed):
    g = torch.Generator().manual_seed(seed)
    mag = torch.exp(torch.randn(layers, 2, hkv, 1, 128, generator=g) * 2)
    x = (torch.randn(layers, 2, hkv, rows, 128, generator=g) * mag).to(torch.bfloat16).to(dev)
    kv8, planes = _cache(dev, list(x.flatten(0, 1)), capacity)
    kv8.seal(planes, 64)
    if rows > 64:
        kv8.seal(planes, rows - 64)   # the next rows, from the row of the same number
    assert kv8.sealed == rows
    kv8.raise_on_device_error()
    _check(kv8, x, 0, rows)
    if capacity > rows:  # unused blocks untouched
        assert not kv8.data[:, :, :, rows:].any() and bool((kv8.scale[..., rows // 64:] == 1).all())
    # any row range back, at another offset; other rows untouched
    from hsd_b200.compaction import plane_pointers
    back = torch.full((layers, 2, hkv, rows + 9, 128), 7.0, dtype=torch.bfloat16, device=dev)
    bp = plane_pointers(list(back.flatten(0, 1)))
    lo, hi = 5, rows - 3
    kv8.unseal(bp, lo, hi - lo, dst_row0=lo + 9)
    want = (kv8.data[:, :, :, :rows].float()
            * kv8.scale[..., :rows // 64].repeat_interleave(64, -1)[..., None]).to(torch.bfloat16)
    assert torch.equal(back[:, :, :, lo + 9:hi + 9], want[:, :, :, lo:hi])
    assert bool((back[:, :, :, :lo + 9] == 7).all()) and bool((back[:, :, :, hi + 9:] == 7).all())


def test_every_pair_of_bf16_significands_rounds_correctly(dev):
    """a / b over all 8-bit significands, exponents 0..9 apart, both signs:
    exact ties and the nearest misses included."""
    sig = torch.arange(128, 256).float()
    blocks = []
    for b in range(128, 256):          # the block's maximum
        vals = torch.cat([sig * 2.0 ** -e for e in range(0, 10)])
        vals = vals[vals <= b]
        body = torch.zeros(64 * 128)
        body[:vals.numel()] = vals
        body[vals.numel():2 * vals.numel()] = -vals
        body[-1] = b
        blocks.append(body.view(64, 128))
    x = torch.cat(blocks)[None].to(torch.bfloat16)          # [1, 8192, 128]
    both = torch.stack([x, x * 2.0 ** 40])[None].to(dev)     # K and V plane
    kv8, planes = _cache(dev, [both[0, 0], both[0, 1]], x.shape[1])
    kv8.seal(planes, x.shape[1])
    _check(kv8, both, 0, x.shape[1])


def test_zero_tiny_and_huge_blocks(dev):
    x = torch.zeros(1, 2, 1, 256, 128)
    x[0, 0, 0, 64:128] = 1e-39            # bf16 subnormals: below 2^-100, held as zeros
    x[0, 0, 0, 128:192] = 3.3e38
    x[0, 0, 0, 192:, ::2] = 2.0 ** -99
    x[0, 1, 0, 3, 7] = -1.0
    x = x.to(torch.bfloat16).to(dev)
    kv8, planes = _cache(dev, [x[0, 0], x[0, 1]], 256)
    kv8.seal(planes, 256)
    kv8.raise_on_device_error()
    _check(kv8, x, 0, 256)
    assert bool((kv8.scale > 0).all())


def test_infinities_and_nan_are_reported(dev):
    from hsd_b200 import _native as N
    g = torch.Generator().manual_seed(4)
    x = torch.randn(1, 2, 1, 192, 128, generator=g).to(torch.bfloat16)
    x[0, 0, 0, 70, 3] = float("inf")
    x[0, 0, 0, 71, 4] = -float("inf")
    x[0, 1, 0, 130, 127] = float("nan")
    x = x.to(dev)
    kv8, planes = _cache(dev, [x[0, 0], x[0, 1]], 192)
    kv8.seal(planes, 192)
    _check(kv8, x, 0, 192)
    assert int(kv8.data[0, 0, 0, 70, 3]) == 127 and int(kv8.data[0, 0, 0, 71, 4]) == -127
    assert int(kv8.data[0, 1, 0, 130, 127]) == 0
    with pytest.raises(N.HSDError, match="infinity"):
        kv8.raise_on_device_error()


def test_replayed_graph_seals_what_the_planes_hold_then(dev):
    x = torch.zeros(1, 2, 2, 64, 128, dtype=torch.bfloat16, device=dev)
    kv8, planes = _cache(dev, [x[0, 0], x[0, 1]], 64)
    kv8.seal(planes, 64)
    kv8.reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.seal(planes, 64)
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        _check(kv8, x, 0, 64)


def test_offsets_past_32_bits(dev):
    """The last plane of a cache of more than 2^31 bytes."""
    from hsd_b200.compaction import plane_pointers
    from hsd_b200.kv8 import Kv8Cache
    cap = 9 * 2 ** 20                     # 9 M rows x 128 = 1.2e9 bytes a plane
    kv8 = Kv8Cache(1, 1, cap, device=dev)
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 1, 128, 128, generator=g).to(torch.bfloat16).to(dev)
    kv8.sealed = cap - 128
    kv8.seal(plane_pointers([x[0], x[1]]), 128, src_row0=0)
    n, s = OK.seal(x.cpu())
    assert np.array_equal(kv8.data[0, :, :, -128:].cpu().numpy(), n)
    assert np.array_equal(kv8.scale[0, :, :, -2:].cpu().numpy(), s.astype(np.float32))
    assert not kv8.data[0, :, :, -192:-128].any()
    back = torch.zeros_like(x)
    kv8.unseal(plane_pointers([back[0], back[1]]), cap - 100, 100, dst_row0=28)
    want = (torch.from_numpy(n).float() * torch.from_numpy(s.astype(np.float32)).repeat_interleave(
        64, -1)[..., None]).to(torch.bfloat16).to(dev)
    assert torch.equal(back[:, :, 28:], want[:, :, 28:]) and not back[:, :, :28].any()
