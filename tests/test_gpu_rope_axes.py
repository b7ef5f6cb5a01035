"""GPU parity of the rotary embedding with several position axes.

Against 64-bit angles and products (``oracle/rope_axes.py``).  Tolerance, from
the arithmetic: the angle reaches the cosine and sine in fp32 (2^-25 half
turns, at most 2^-23 rad), they are off by a further 2^-23 at most, so a
value is off by 2^-21 (|x_i| + |x_{i+64}|) before its one rounding to bf16,
half a step: 2^-8 of the value.
"""
import numpy as np
import pytest
import torch

from oracle import rope_axes as OA

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from hsd_b200 import _native
    _native.load()
    return torch.device("cuda:0")


def _check(got, x, pos, sections, interleaved=False, theta=1e6, scaling=1.0, inv_freq=None):
    """got / x: [rows, heads, 128]"""
    freq = inv_freq if inv_freq is not None else [theta ** (-i / 64) for i in range(64)]
    x = x.double().cpu().numpy()
    want = OA.rotate(x, pos.cpu().numpy(), OA.pair_axis(sections, interleaved), freq, scaling)
    mag = np.abs(x[..., :64]) + np.abs(x[..., 64:])
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -21 * abs(scaling) * np.concatenate([mag, mag], -1)
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("n,hq,hkv,sections,interleaved,far,theta", [
    (1, 16, 8, [16, 16, 16, 16], False, 5000, 1e6),       # one token, the HunYuan split
    (1, 1, 1, [64], False, 3, 1e4),                        # one axis, one head
    (37, 12, 2, [16, 24, 24], False, 6000, 1e6),
    (129, 12, 2, [24, 20, 20], True, 131072, 1e6),         # far positions
    (700, 5, 1, [1, 62, 1], False, 1 << 40, 5e5),          # positions past 32 bits
    (1300, 28, 4, [0, 64], False, 100, 1e4),               # an axis without pairs
    (593, 4, 4, [8] * 8, True, 50, 1e6),                   # eight axes
])
def test_matches_64_bit_formula(dev, n, hq, hkv, sections, interleaved, far, theta):
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    g = torch.Generator().manual_seed(n + hq)
    w = (hq + 2 * hkv) * 128
    qkv = (torch.randn(n, w, generator=g) * 2).to(torch.bfloat16).to(dev)
    pos = torch.randint(-far, far, (len(sections), n), generator=g).to(dev)
    row0, cap = 11, n + 13
    kc = torch.randn(hkv, cap, 128, generator=g).to(torch.bfloat16).to(dev)
    vc = torch.randn(hkv, cap, 128, generator=g).to(torch.bfloat16).to(dev)
    kc0, vc0, qkv0 = kc.clone(), vc.clone(), qkv.clone()
    rot = RotaryAxes(sections, theta=theta, interleaved=interleaved, device=dev)
    a, b = hq * 128, (hq + hkv) * 128
    q = rope_append_axes(qkv[:, :a], qkv[:, a:b], qkv[:, b:], pos, rot, kc, vc, row0)
    torch.cuda.synchronize()
    assert q.shape == (1, hq, n, 128) and q.data_ptr() == qkv.data_ptr()
    x = qkv0.view(n, hq + 2 * hkv, 128)
    args = (pos, sections, interleaved, theta)
    _check(q[0].transpose(0, 1), x[:, :hq], *args)
    _check(kc[:, row0:row0 + n].transpose(0, 1), x[:, hq:hq + hkv], *args)
    assert torch.equal(vc[:, row0:row0 + n].transpose(0, 1), x[:, hq + hkv:])
    # nothing else was written
    assert torch.equal(qkv[:, a:], qkv0[:, a:])
    for c, c0 in ((kc, kc0), (vc, vc0)):
        assert torch.equal(c[:, :row0], c0[:, :row0]) and torch.equal(c[:, row0 + n:],
                                                                      c0[:, row0 + n:])


def test_positions_layouts_out_and_scaling(dev):
    """[1, A, Q] and [A, 1, Q] ids, an expanded row, int32, rotation into out
    (q kept), keys and values only, a model's own fp32 frequencies, scaling."""
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    g = torch.Generator().manual_seed(3)
    n, hq, hkv = 50, 6, 2
    q = torch.randn(n, hq * 128, generator=g).to(torch.bfloat16).to(dev)
    k = torch.randn(n, hkv * 128, generator=g).to(torch.bfloat16).to(dev)
    v = torch.randn(n, 3 * hkv * 128, generator=g).to(torch.bfloat16).to(dev)[:, :hkv * 128]
    inv = (1.0 / 1e4 ** (torch.arange(0, 128, 2).float() / 128))
    rot = RotaryAxes([16, 16, 16, 16], inv_freq=inv, scaling=1.25, device=dev)
    one = torch.randint(0, 9000, (n,), generator=g).to(dev)
    kc = torch.zeros(1, hkv, n, 128, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    q0 = q.clone()
    base = None
    for pos in (one[None, None].expand(1, 4, n), one[None, None].expand(4, 1, n),
                one[None].repeat(4, 1).int()):
        out = torch.empty(n, hq * 128 + 64, dtype=torch.bfloat16, device=dev)[:, :hq * 128]
        r = rope_append_axes(q, k, v, pos, rot, kc, vc, 0, out=out)
        assert torch.equal(q, q0) and r.data_ptr() == out.data_ptr()
        if base is None:
            base = (r.clone(), kc.clone())
            _check(r[0].transpose(0, 1), q0.view(n, hq, 128), one[None].repeat(4, 1),
                   [16] * 4, scaling=1.25, inv_freq=[float(f) for f in inv])
        assert torch.equal(r, base[0]) and torch.equal(kc, base[1])
    kc.zero_()
    assert rope_append_axes(None, k, v, pos, rot, kc, vc, 0) is None
    assert torch.equal(kc, base[1])
    assert torch.equal(vc[0].transpose(0, 1).reshape(n, -1), v)


def test_zero_rows_and_side_stream(dev):
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    rot = RotaryAxes([64], device=dev)
    kc = torch.ones(2, 8, 128, dtype=torch.bfloat16, device=dev)
    e = torch.empty(0, 256, dtype=torch.bfloat16, device=dev)
    r = rope_append_axes(e, e, e, torch.empty(1, 0, dtype=torch.int64, device=dev), rot, kc,
                         kc.clone(), 8)
    assert r.shape == (1, 2, 0, 128) and bool((kc == 1).all())
    # position 0 on another stream: a copy
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.randn(3, 256, device=dev).to(torch.bfloat16)
        y = x.clone()
        vc = torch.zeros_like(kc)
        rope_append_axes(y, x, x, torch.zeros(1, 3, dtype=torch.int64, device=dev), rot, kc, vc, 5)
    s.synchronize()
    assert torch.equal(x, y)
    assert torch.equal(kc[:, 5:].transpose(0, 1).reshape(3, 256), x)


def test_graph_replay_reads_new_positions(dev):
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    rot = RotaryAxes([32, 32], device=dev)
    n = 9
    x = torch.randn(n, 256, device=dev).to(torch.bfloat16)
    out, kc, vc = torch.empty_like(x), torch.zeros(2, n, 128, dtype=torch.bfloat16, device=dev), \
        torch.zeros(2, n, 128, dtype=torch.bfloat16, device=dev)
    pos = torch.zeros(2, n, dtype=torch.int64, device=dev)
    rope_append_axes(x, x, x, pos, rot, kc, vc, 0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rope_append_axes(x, x, x, pos, rot, kc, vc, 0, out=out)
    pos.copy_(torch.arange(2 * n, device=dev).view(2, n))
    graph.replay()
    torch.cuda.synchronize()
    _check(out.view(n, 2, 128), x.view(n, 2, 128), pos, [32, 32])
    assert torch.equal(kc.transpose(0, 1).reshape(n, 256), out)


def test_bad_pair_axis_is_reported(dev):
    """A table entry outside the axes is refused by the kernel's own check."""
    from hsd_b200 import _native as N
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    rot = RotaryAxes([64], device=dev)
    rot.pair_axis[5] = 7
    x = torch.randn(2, 128, device=dev).to(torch.bfloat16)
    y = x.clone()
    kc = torch.zeros(1, 2, 128, dtype=torch.bfloat16, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    rope_append_axes(y, x, x, torch.ones(1, 2, dtype=torch.int64, device=dev), rot, kc,
                     kc.clone(), 0, status=st)
    assert int(st.item()) & N.HSD_DEV_BAD_INDEX
    assert torch.equal(y[:, [5, 69]], x[:, [5, 69]]) and not torch.equal(y[:, 4], x[:, 4])


def test_cache_offsets_past_32_bits(dev):
    """The last head's rows of caches of more than 2^31 elements."""
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    rot = RotaryAxes([64], device=dev)
    kc = torch.empty(2, 9 * 2 ** 20, 128, dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    n = 5
    row0 = kc.shape[1] - n
    x = torch.randn(n, 256, device=dev).to(torch.bfloat16)
    rope_append_axes(None, x, x, torch.zeros(1, n, dtype=torch.int64, device=dev), rot, kc, vc,
                     row0)
    for c in (kc, vc):
        assert torch.equal(c[:, row0:].transpose(0, 1).reshape(n, 256), x)


def test_refusals(dev):
    """Every refusal of the binding, on real tensors; nothing is launched."""
    from hsd_b200 import _native as N
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    rot = RotaryAxes([32, 32], device=dev)
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=dev)
    kc = torch.zeros(2, 8, 128, dtype=torch.bfloat16, device=dev)
    pos = torch.zeros(2, 4, dtype=torch.int64, device=dev)
    ok = dict(q=x, k=x.clone(), v=x.clone(), positions=pos, rotary=rot, k_cache=kc,
              v_cache=kc.clone(), dst_row0=4)
    bad = [
        dict(q=x.float()), dict(q=x[:3]), dict(q=x[:, :200]), dict(q=x.cpu()), dict(k=x[:3]),
        dict(k=x[:, :128]), dict(v=x[:3]), dict(k=x.t().contiguous().t()), dict(positions=pos[:1]),
        dict(positions=pos[:, :3]), dict(positions=pos.float()), dict(positions=pos.cpu()),
        dict(positions=pos[None, None]), dict(dst_row0=5), dict(dst_row0=-1),
        dict(k_cache=kc[:1]), dict(k_cache=kc.float()), dict(k_cache=kc.cpu()),
        dict(k_cache=kc[:, :, :64]), dict(v_cache=torch.zeros(2, 9, 128, dtype=torch.bfloat16,
                                                             device=dev)),
        dict(q=None, out=x), dict(out=x[:3]), dict(out=x.float()), dict(num_q_heads=3),
        dict(num_kv_heads=1), dict(rotary=RotaryAxes([32, 32], device="cpu")),
        dict(status=torch.zeros(1, device=dev)),
        dict(out=torch.zeros(256, 4, dtype=torch.bfloat16, device=dev).t()),
    ]
    for change in bad:
        with pytest.raises((ValueError, TypeError, N.HSDError)):
            rope_append_axes(**{**ok, **change})
    assert not kc.any()
    rope_append_axes(**ok)
    torch.cuda.synchronize()
