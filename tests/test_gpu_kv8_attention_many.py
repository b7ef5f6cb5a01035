"""The 8-bit attention's path for many rows (expansion + scaled tcgen05 kernel),
the border between the two paths, and what both have to survive.

Oracle and tolerances: ``tests/test_gpu_kv8_attention.py``.
"""
import math

import pytest
import torch

from tests import test_gpu_kv8_attention as T

pytestmark = pytest.mark.gpu
dev = T.dev


def many(q_len, kv_len, hq, hkv):
    """Whether these sizes take the path for many rows (its workspace holds the
    layer's columns)."""
    from hsd_b200 import _native as N
    return N.load().hsd_kv8_attention_workspace_bytes(q_len, kv_len, hq, hkv) \
        >= 512 * hkv * kv_len


@pytest.mark.parametrize("lens,pad,prefix,sealed,hq,hkv", [
    ([700], 0, 640, 640, 12, 2),                      # everything in front sealed
    ([700, 1, 333], 118, 1100, 1088, 12, 2),          # padded rows, a bf16 remainder
    ([900], 0, 700, 0, 5, 1),                         # bf16 alone, odd heads
    ([1500], 0, 130, 64, 4, 4),                       # one query head per KV head
    ([61, 34, 118, 47, 300, 25, 90, 63, 55, 140, 38, 81, 60, 29, 104, 66], 0, 1600, 1600, 16, 8),
    ([1025], 0, 63, 0, 28, 4),                        # no whole block in front
    ([513] * 3, 5, 257, 192, 6, 2),
    ([2300], 0, 700, 0, 5, 1),
    ([2000], 0, 130, 64, 4, 4),
])
def test_segments(dev, lens, pad, prefix, sealed, hq, hkv):
    allowed = T.segments(lens, prefix, pad).to(dev)
    q_len, kv_len = allowed.shape
    assert many(q_len, kv_len, hq, hkv) or (q_len, hq) == (900, 5)   # few enough rows there
    x = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=prefix)
    want = T.exact(*x, sealed, allowed)
    plan = T.plan_of(allowed)
    a = T.run(*x, sealed, plan)
    T.check(a, want)
    b = T.run(*x, sealed, plan, tail_row0=sealed)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("q_len", [16, 64, 200, 400, 900])
def test_both_sides_of_the_choice_agree(dev, q_len):
    """The same rows alone (few rows) and as part of a longer query (many)."""
    hq, hkv, kv_len, sealed = 12, 2, 3000, 2944
    x = T.make(dev, hq, hkv, 1000, kv_len, sealed, seed=q_len)
    allowed = T.segments([1000], kv_len - 1000).to(dev)
    assert many(1000, kv_len, hq, hkv)
    full = T.run(*x, sealed, T.plan_of(allowed))
    part = (x[0][:, :q_len].contiguous(),) + x[1:]
    a = allowed[:q_len]
    got = T.run(*part, sealed, T.plan_of(a))
    want = T.exact(*part, sealed, a)
    T.check(got, want)
    # two roundings of the same value: half a step each, and P's (2^-11, sealed columns)
    tol = 2.0 ** -7 * want[0].abs() + 2.0 ** -9 * want[2].t()[..., None]
    assert ((got[0].double() - full[0][:q_len].double()).abs() <= tol).all()


@pytest.mark.parametrize("hq,density,seed", [(6, 0.5, 0), (6, 0.01, 1), (12, 0.3, 3),
                                             (12, 0.005, 4), (12, 0.0, 2), (2, 0.5, 5),
                                             (2, 0.01, 6)])
def test_random_masks_and_empty_rows(dev, hq, density, seed):
    q_len, kv_len, sealed, hkv = 800, 1300, 640, 2
    g = torch.Generator().manual_seed(seed)
    allowed = torch.rand(q_len, kv_len, generator=g) < density
    allowed[::3] = False
    allowed[128:256] = False              # a query tile that sees nothing
    allowed[:, 64:300] = False            # column tiles that nobody sees
    allowed = allowed.to(dev)
    assert many(q_len, kv_len, hq, hkv) == (hq > 2)
    x = T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=seed)
    T.check(T.run(*x, sealed, T.plan_of(allowed)), T.exact(*x, sealed, allowed))


def test_masked_columns_may_hold_anything(dev):
    q_len, kv_len, sealed, hq, hkv = 900, 1200, 192, 8, 2
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed)
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    for lo, hi in ((200, 230), (300, 450), (1190, 1200)):
        allowed[:, lo:hi] = False
    tail[:, :, 200:230] = float("nan")
    tail[:, :, 300:450] = float("inf")
    tail[:, :, 1190:] = -float("inf")
    tail[:, :, :sealed] = float("nan")
    data[:, :, sealed:] = 99
    scale[:, :, sealed // 64:] = float("nan")
    assert many(q_len, kv_len, hq, hkv)
    T.check(T.run(q, data, scale, tail, sealed, T.plan_of(allowed)),
            T.exact(q, data, scale, tail, sealed, allowed))


@pytest.mark.parametrize("q_len", [3, 40, 900, 2500])
def test_values_of_unlike_magnitude(dev, q_len):
    """V blocks from 2^-30 to 2^30 of each other, sealed and bf16; rows that see
    only one of them."""
    kv_len, sealed, hq, hkv = 1024, 512, 6, 2
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed)
    mag = torch.exp2(torch.linspace(-30, 30, 16, device=dev))[torch.randperm(
        16, generator=torch.Generator().manual_seed(1)).to(dev)]
    scale[1] = torch.cat([mag[:8], mag[:1]])[None] / 70
    tail[1] = (tail[1].float() * mag.repeat_interleave(64)[None, :, None]).to(torch.bfloat16)
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    for r in range(1, q_len):
        if r % 3:
            allowed[r] = False
            b = r % 16
            allowed[r, 64 * b:64 * b + 64] = True
    T.check(T.run(q, data, scale, tail, sealed, T.plan_of(allowed)),
            T.exact(q, data, scale, tail, sealed, allowed))


@pytest.mark.parametrize("q_len", [2, 30, 900, 2500])
def test_blocks_of_zeros(dev, q_len):
    """Sealed blocks of zeros (scale 2^-100 / 127) among others, whole caches of
    zeros, and a bf16 tail of zeros: weights count, values are 0."""
    from hsd_b200.kv8 import Kv8Cache
    from hsd_b200.compaction import plane_pointers
    hq, hkv, kv_len, sealed = 6, 2, 800, 512
    g = torch.Generator(device=dev).manual_seed(0)
    q = torch.randn(hq, q_len, 128, generator=g, device=dev).to(torch.bfloat16)
    kv = torch.randn(2, hkv, kv_len, 128, generator=g, device=dev).to(torch.bfloat16)
    kv[0, :, 64:192] = 0
    kv[1, :, 128:320] = 0
    kv[1, 0] = 0
    kv[:, :, 700:] = 0
    kv8 = Kv8Cache(1, hkv, 576, device=dev)
    kv8.seal(plane_pointers([kv[0], kv[1]]), sealed)
    kv8.raise_on_device_error()
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    data, scale = kv8.data[0], kv8.scale[0]
    got = T.run(q, data, scale, kv, sealed, T.plan_of(allowed))
    want = T.exact(q, data, scale, kv, sealed, allowed)
    T.check(got, want)
    assert bool((got[0][:, :3] == 0).all())     # the head whose values are all zeros


@pytest.mark.parametrize("q_len", [1, 9, 700, 2500])
def test_large_scores_between_blocks(dev, q_len):
    """Scores that jump by hundreds between blocks, up and down, and one row
    whose scores are all far below the others'."""
    kv_len, sealed, hq, hkv = 900, 640, 4, 2
    q, data, scale, tail = T.make(dev, hq, hkv, q_len, kv_len, sealed)
    jump = torch.tensor([1, 40, 3, 200, 5, 90, 1, 300, 2, 60, 1], device=dev).float()
    scale[0] = jump[None] / 70
    tail[0] *= 30
    q[:, -1] *= 0.01
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    got = T.run(q, data, scale, tail, sealed, T.plan_of(allowed))
    want = T.exact(q, data, scale, tail, sealed, allowed)
    T.check(got, want)


def test_streams_and_graphs_share_nothing(dev):
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    hq, hkv = 12, 2
    cases = []
    for i, ln in enumerate(([900], [300, 500, 41])):
        allowed = T.segments(ln, 1500).to(dev)
        q_len, kv_len = allowed.shape
        assert many(q_len, kv_len, hq, hkv)
        x = T.make(dev, hq, hkv, q_len, kv_len, 1472, seed=i)
        plan = T.plan_of(allowed)
        cases.append((x, plan, T.run(*x, 1472, plan)))

    def call(x, plan):
        return verify_attention_kv8(x[0], Kv8Layer(x[1][0], x[1][1], x[2][0], x[2][1]), 1472,
                                    x[3][0], x[3][1], plan)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for (x, plan, _), s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(call(x, plan))
        torch.cuda.synchronize()
        for (o, l), (_, _, w) in zip(got, cases):
            assert torch.equal(o, w[0]) and torch.equal(l, w[1])
    graphs = []
    for x, plan, _ in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a = call(x, plan)
            b = call(x, plan)       # two calls of one graph
        graphs.append((graph, a, b))
    for _ in range(4):
        for (graph, _, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, a, b), (_, _, w) in zip(graphs, cases):
            for o, l in (a, b):
                assert torch.equal(o, w[0]) and torch.equal(l, w[1])
                o.zero_()
                l.zero_()
        torch.cuda.synchronize()


def test_repeated_calls_are_bitwise_equal(dev):
    for lens, kv in (([1], 20000), ([1] * 33, 5000), ([1200], 4000)):
        allowed = T.segments(lens, kv).to(dev)
        x = T.make(dev, 16, 8, allowed.shape[0], allowed.shape[1], kv // 64 * 64, seed=kv)
        plan = T.plan_of(allowed)
        a = T.run(*x, kv // 64 * 64, plan)
        for _ in range(3):
            b = T.run(*x, kv // 64 * 64, plan)
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_long_cache(dev):
    """A hundred thousand columns, one row and a few (more CTAs than a cluster,
    joined by the second launch), against 64 bits."""
    for lens, hq, hkv in (([1], 8, 1), ([1, 2], 12, 2), ([17], 4, 2)):
        prefix = 100_003
        allowed = T.segments(lens, prefix).to(dev)
        sealed = prefix // 64 * 64
        x = T.make(dev, hq, hkv, allowed.shape[0], allowed.shape[1], sealed, seed=1)
        T.check(T.run(*x, sealed, T.plan_of(allowed)), T.exact(*x, sealed, allowed))


def test_out_and_lse_given(dev):
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    for q_len in (2, 900, 2500):
        q, data, scale, tail = T.make(dev, 6, 2, q_len, 700, 640)
        allowed = torch.ones(q_len, 700, dtype=torch.bool, device=dev)
        plan = T.plan_of(allowed)
        out = torch.empty(q_len, 6, 128, dtype=torch.bfloat16, device=dev)
        lse = torch.empty(6, q_len, device=dev)
        o, l = verify_attention_kv8(q, Kv8Layer(data[0], data[1], scale[0], scale[1]), 640, tail[0],
                                    tail[1], plan, out=out, lse=lse, scale=0.05)
        assert o.data_ptr() == out.data_ptr() and l.data_ptr() == lse.data_ptr()
        T.check((o, l), T.exact(q, data, scale, tail, 640, allowed, sm=0.05))


def test_refusals(dev):
    """Every refusal of the binding, on real tensors; nothing is launched."""
    from hsd_b200 import _native as N
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    q, data, scale, tail = T.make(dev, 6, 2, 10, 700, 640)
    plan = T.plan_of(torch.ones(10, 700, dtype=torch.bool, device=dev))
    layer = Kv8Layer(data[0], data[1], scale[0], scale[1])
    ok = dict(q=q, layer=layer, sealed=640, k=tail[0], v=tail[1], plan=plan)
    bad = [
        dict(q=q.float()), dict(q=q[:, :9]), dict(q=q[..., :64]), dict(q=q[:5]), dict(q=q.cpu()),
        dict(q=q[None].expand(2, -1, -1, -1)), dict(sealed=639), dict(sealed=-64),
        dict(sealed=704), dict(layer=None), dict(layer=layer[:3]), dict(k=None),
        dict(k=tail[0][:, :100]), dict(v=tail[1][:1]), dict(k=tail[0].float()), dict(k=tail[0].cpu()),
        dict(tail_row0=641), dict(tail_row0=-1), dict(scale=0.0), dict(scale=-1.0),
        dict(scale=math.inf), dict(scale=math.nan),
        dict(layer=Kv8Layer(data[0].float(), data[1], scale[0], scale[1])),
        dict(layer=Kv8Layer(data[0][:, :600], data[1], scale[0], scale[1])),
        dict(layer=Kv8Layer(data[0].transpose(0, 1), data[1], scale[0], scale[1])),
        dict(layer=Kv8Layer(data[0], data[1], scale[0][:, :9], scale[1])),
        dict(layer=Kv8Layer(data[0], data[1], scale[0].double(), scale[1])),
        dict(layer=Kv8Layer(data[0].cpu(), data[1], scale[0], scale[1])),
        dict(out=torch.empty(10, 6, 128, device=dev)), dict(lse=torch.empty(6, 9, device=dev)),
        dict(k=tail[0].expand(2, -1, -1)[:1].expand(2, -1, -1)),   # heads of stride 0
    ]
    for change in bad:
        with pytest.raises((ValueError, TypeError, N.HSDError)):
            verify_attention_kv8(**{**ok, **change})
    out, lse = verify_attention_kv8(**ok)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("q_len", [1, 5])
@pytest.mark.parametrize("kv_len", [130, 600, 1100, 1600, 2100, 2600, 3100, 3600, 4100, 9000])
def test_splits_of_few_rows(dev, q_len, kv_len):
    """3 and 15 packed rows over ever more columns: one CTA, clusters of each size,
    and more CTAs than a cluster holds."""
    sealed = (kv_len - 40) // 64 * 64
    allowed = T.segments([q_len], kv_len - q_len).to(dev)
    x = T.make(dev, 6, 2, q_len, kv_len, sealed, seed=kv_len)
    T.check(T.run(*x, sealed, T.plan_of(allowed)), T.exact(*x, sealed, allowed))


@pytest.mark.parametrize("q_len", [3, 900])
def test_plan_rebuilt_in_a_graph(dev, q_len):
    """One graph builds the plan of a mask and attends in two layers right behind
    it; replayed with other masks in the same memory."""
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    from hsd_b200.plan import plan_from_dense
    hq, hkv, kv_len, sealed = 12, 2, 2000, 1024
    assert many(q_len, kv_len, hq, hkv) == (q_len == 900)
    layers = [T.make(dev, hq, hkv, q_len, kv_len, sealed, seed=s) for s in (1, 2)]
    g = torch.Generator().manual_seed(3)
    masks, want = [], []
    for density in (0.5, 0.02, 1.0, 0.0):
        allowed = (torch.rand(q_len, kv_len, generator=g) < density).to(dev)
        masks.append(torch.where(allowed, 0.0, -math.inf))
        want.append([T.run(*x, sealed, T.plan_of(allowed)) for x in layers])
    mask = masks[2].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan = plan_from_dense(mask)
        got = [verify_attention_kv8(x[0], Kv8Layer(x[1][0], x[1][1], x[2][0], x[2][1]), sealed,
                                    x[3][0], x[3][1], plan) for x in layers]
    for i in (0, 1, 2, 3, 1, 0):
        mask.copy_(masks[i])
        graph.replay()
        torch.cuda.synchronize()
        plan.raise_on_device_error()
        for (o, l), (wo, wl) in zip(got, want[i]):
            assert torch.equal(o, wo) and torch.equal(l, wl)
