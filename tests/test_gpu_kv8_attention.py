"""GPU parity of the attention over the 8-bit cache, against 64 bits.

Tolerance, from the arithmetic.  P is rounded (or truncated, with the bias
taken out) to bf16, at most 2^-7 of each weight; the output is a weighted
mean of V, so it is off by at most 2^-7 max|V| over the row's visible columns,
plus half a bf16 step (2^-8) of itself and of joined partial rows.  Errors of
independent weights cancel, so the RMS error is held far lower: 2^-8 of the
outputs' RMS for P and 2^-8 for each rounding of the output.  Scores: fp32
sums of 128 products and exponentials, 2^-18 of the largest |score| for the
lse, plus its own rounding.
"""
import math

import numpy as np
import pytest
import torch

from oracle import masks as OM

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    from hsd_b200 import _native
    _native.load()
    return torch.device("cuda:0")


def make(dev, hq, hkv, q_len, kv_len, sealed, seed=0, mag=0.3):
    g = torch.Generator(device=dev).manual_seed(seed)

    def rnd(*s):
        return torch.randn(*s, generator=g, device=dev)
    q = rnd(hq, q_len, 128).to(torch.bfloat16)
    cap = sealed + 64          # a block more than is in use
    data = torch.randint(-127, 128, (2, hkv, cap, 128), generator=g, device=dev,
                         dtype=torch.int8)
    scale = torch.exp(rnd(2, hkv, cap // 64) * mag) / 70
    tail = rnd(2, hkv, kv_len, 128).to(torch.bfloat16)
    return q, data, scale, tail


def exact(q, data, scale, tail, sealed, allowed, sm=None):
    """64 bits; columns that no row sees do not matter."""
    hq, q_len, _ = q.shape
    hkv, kv_len = tail.shape[1], allowed.shape[1]
    sm = 1 / math.sqrt(128) if sm is None else sm
    kv = torch.cat([data[:, :, :sealed].double()
                    * scale[..., :sealed // 64].double().repeat_interleave(64, -1)[..., None],
                    tail[:, :, sealed:kv_len].double()], 2)
    seen = allowed.any(0)
    kv = torch.where(seen[None, None, :, None], kv, 0.0)
    out = torch.empty(q_len, hq, 128, dtype=torch.float64, device=q.device)
    lse = torch.empty(hq, q_len, dtype=torch.float64, device=q.device)
    bound = torch.empty(hq, q_len, dtype=torch.float64, device=q.device)
    top = 0.0
    for h in range(hq):
        k, v = kv[0, h * hkv // hq], kv[1, h * hkv // hq]
        s = (q[h].double() @ k.t()) * sm
        top = max(top, float(s.abs().max()))
        s = s.masked_fill(~allowed, -math.inf)
        lse[h] = torch.logsumexp(s, -1)
        p = torch.nan_to_num(torch.exp(s - lse[h][:, None]), nan=0.0)
        out[:, h] = p @ v
        bound[h] = (allowed.double() * v.abs().amax(-1)[None]).amax(-1)
    return out, lse, bound, top


def check(got, want):
    out, lse = got
    w_out, w_lse, vmax, top = want
    out = out.double()
    assert torch.isfinite(out).all()
    err = (out - w_out).abs()
    tol = 2.0 ** -7 * vmax.t()[..., None] + 2.0 ** -7 * w_out.abs()
    assert (err <= tol).all(), float((err - tol).max())
    rms = w_out.pow(2).mean().sqrt()
    assert err.pow(2).mean().sqrt() <= 3 * 2.0 ** -8 * rms + 1e-30
    empty = torch.isinf(w_lse)
    assert torch.equal(torch.isinf(lse), empty) and bool((lse[empty] < 0).all())
    assert bool((out[empty.t()] == 0).all())
    err = (lse.double() - w_lse)[~empty].abs()
    if err.numel():
        assert float(err.max()) <= 2.0 ** -18 * (top + float(w_lse[~empty].abs().max()) + 1)


def plan_of(allowed):
    from hsd_b200.plan import plan_from_dense
    m = torch.where(allowed, 0.0, -math.inf)
    return plan_from_dense(m)


def run(q, data, scale, tail, sealed, plan, tail_row0=0, **kw):
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    layer = Kv8Layer(data[0], data[1], scale[0], scale[1])
    t = tail[:, :, tail_row0:]
    got = verify_attention_kv8(q, layer, sealed, t[0], t[1], plan, tail_row0=tail_row0, **kw)
    torch.cuda.synchronize()
    plan.raise_on_device_error()
    return got


def segments(lens, prefix, pad=0):
    """allowed of causal segments behind a prefix that all see"""
    q_len = sum(lens) + pad
    a = torch.zeros(q_len, prefix + q_len, dtype=torch.bool)
    at = 0
    for n in lens:
        a[at:at + n, :prefix] = True
        a[at:at + n, prefix + at:prefix + at + n] = torch.ones(n, n, dtype=torch.bool).tril()
        at += n
    return a


CASES = [
    # lens, pad, prefix, sealed, hq, hkv
    ([1], 0, 64, 64, 12, 2),
    ([1], 0, 1, 0, 1, 1),                 # two columns, nothing sealed
    ([1], 0, 2624, 2560, 12, 2),          # a token; 64 prompt columns in bf16
    ([1], 0, 5000, 4992, 16, 8),
    ([1] * 40, 0, 700, 640, 12, 2),
    ([3, 1, 7], 5, 200, 128, 5, 1),       # odd heads, padded rows
    ([17], 0, 130, 0, 4, 4),              # bf16 alone
    ([64, 96, 128, 200], 24, 1024, 1024, 12, 2),
    ([61, 34, 118, 1, 72], 98, 1600, 1536, 16, 8),
    ([129], 0, 63, 0, 8, 1),
    ([300], 0, 640, 640, 28, 4),
    ([2, 255], 0, 1000, 64, 6, 2),        # a long bf16 tail
]


@pytest.mark.parametrize("lens,pad,prefix,sealed,hq,hkv", CASES)
def test_segments(dev, lens, pad, prefix, sealed, hq, hkv):
    allowed = segments(lens, prefix, pad).to(dev)
    x = make(dev, hq, hkv, allowed.shape[0], allowed.shape[1], sealed, seed=prefix)
    want = exact(*x, sealed, allowed)
    plan = plan_of(allowed)
    a = run(*x, sealed, plan)
    check(a, want)
    b = run(*x, sealed, plan, tail_row0=sealed)   # the rows behind the sealed ones alone
    c = run(*x, sealed, plan, need_lse=False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(a[0], c[0]) and c[1] is None


@pytest.mark.parametrize("q_len,kv_len,sealed,hq,hkv,density,seed", [
    (1, 700, 640, 12, 2, 0.5, 0), (9, 333, 128, 6, 2, 0.02, 1), (150, 513, 512, 4, 2, 0.3, 2),
    (260, 900, 448, 3, 3, 0.003, 3),
])
def test_random_masks_and_empty_rows(dev, q_len, kv_len, sealed, hq, hkv, density, seed):
    g = torch.Generator().manual_seed(seed)
    allowed = torch.rand(q_len, kv_len, generator=g) < density
    allowed[::3] = False
    allowed[:, 64:200] = False            # whole tiles without a column
    allowed = allowed.to(dev)
    x = make(dev, hq, hkv, q_len, kv_len, sealed, seed=seed)
    check(run(*x, sealed, plan_of(allowed)), exact(*x, sealed, allowed))


def test_all_columns_sealed_and_no_tail(dev):
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    for q_len in (3, 200):
        allowed = (torch.rand(q_len, 256, generator=torch.Generator().manual_seed(1)) < 0.7).to(dev)
        q, data, scale, tail = make(dev, 6, 2, q_len, 256, 256)
        got = verify_attention_kv8(q, Kv8Layer(data[0], data[1], scale[0], scale[1]), 256, None,
                                   None, plan_of(allowed))
        check(got, exact(q, data, scale, tail, 256, allowed))


@pytest.mark.parametrize("q_len", [2, 190])
def test_block_scales_of_unlike_size(dev, q_len):
    """Scales 2^-40 to 2^40 between blocks: the softmax may sit on any block,
    and V's scale reaches the output unharmed."""
    q, data, scale, tail = make(dev, 4, 2, q_len, 700, 640)
    e = torch.linspace(-40, 4, 11, device=dev)
    scale[0] = torch.exp2(e.flip(0))[None] / 70
    scale[1] = torch.exp2(e.roll(5) * torch.tensor([[1.0], [-1.0]], device=dev)) / 70
    allowed = torch.ones(q_len, 700, dtype=torch.bool, device=dev)
    allowed[1, :320] = False
    check(run(q, data, scale, tail, 640, plan_of(allowed)), exact(q, data, scale, tail, 640, allowed))


@pytest.mark.parametrize("q_len", [1, 150])
def test_masked_columns_may_hold_anything(dev, q_len):
    kv_len, sealed = 500, 192
    q, data, scale, tail = make(dev, 4, 2, q_len, kv_len, sealed)
    allowed = torch.ones(q_len, kv_len, dtype=torch.bool, device=dev)
    allowed[:, 200:230] = False
    allowed[:, 300:450] = False
    allowed[:, 490:] = False
    tail[:, :, 200:230] = float("nan")
    tail[:, :, 300:450] = float("inf")
    tail[:, :, 490:] = -float("inf")
    tail[:, :, :sealed] = float("nan")     # the sealed rows' bf16 copies are not read
    data[:, :, sealed:] = 99
    scale[:, :, sealed // 64:] = float("nan")
    check(run(q, data, scale, tail, sealed, plan_of(allowed)),
          exact(q, data, scale, tail, sealed, allowed))


@pytest.mark.parametrize("q_len", [5, 140])
def test_strided_inputs(dev, q_len):
    """q as columns of a fused projection, tails as slices of larger caches,
    sealed rows of a cache with room."""
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    hq, hkv, kv_len, sealed = 6, 2, 400, 256
    q, data, scale, tail = make(dev, hq, hkv, q_len, kv_len, sealed)
    allowed = segments([q_len], kv_len - q_len).to(dev)
    want = exact(q, data, scale, tail, sealed, allowed)
    fused = torch.zeros(q_len, (hq + 4) * 128, dtype=torch.bfloat16, device=dev)
    fused[:, :hq * 128] = q.transpose(0, 1).reshape(q_len, -1)
    q2 = fused[:, :hq * 128].unflatten(-1, (hq, 128)).transpose(0, 1)[None]
    room = torch.full((hkv, kv_len + 30, 2, 128), float("nan"), dtype=torch.bfloat16, device=dev)
    room[:, :kv_len] = tail.permute(1, 2, 0, 3)
    big = torch.zeros(hkv, 2, 1024, 128, dtype=torch.int8, device=dev)
    big[:, :, :data.shape[2]] = data.transpose(0, 1)
    sc = torch.full((hkv, 2, 16), float("nan"), device=dev)
    sc[:, :, :scale.shape[2]] = scale.transpose(0, 1)
    layer = Kv8Layer(big[:, 0], big[:, 1], sc[:, 0], sc[:, 1])
    got = verify_attention_kv8(q2, layer, sealed, room[:, :, 0], room[:, :, 1], plan_of(allowed))
    check(got, want)


def test_streams_and_graphs_do_not_share_scratch(dev):
    """Calls on two streams at once, and two graphs captured on one stream and
    replayed on two: every result is the single call's, bit for bit."""
    lens = ([1], [1] * 9, [200, 56])
    cases = []
    for i, ln in enumerate(lens):
        allowed = segments(ln, 3000).to(dev)
        x = make(dev, 12, 2, allowed.shape[0], allowed.shape[1], 2944, seed=i)
        plan = plan_of(allowed)
        cases.append((x, plan, run(*x, 2944, plan)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for x, plan, _ in cases:
            for s in streams:
                with torch.cuda.stream(s):
                    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
                    got.append(verify_attention_kv8(
                        x[0], Kv8Layer(x[1][0], x[1][1], x[2][0], x[2][1]), 2944, x[3][0], x[3][1],
                        plan))
        torch.cuda.synchronize()
        for i, (o, l) in enumerate(got):
            want = cases[i // 2][2]
            assert torch.equal(o, want[0]) and torch.equal(l, want[1])
    graphs = []
    from hsd_b200.kv8 import Kv8Layer, verify_attention_kv8
    for x, plan, _ in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = verify_attention_kv8(x[0], Kv8Layer(x[1][0], x[1][1], x[2][0], x[2][1]), 2944,
                                     x[3][0], x[3][1], plan)
        graphs.append((graph, o))
    for _ in range(5):
        for i, (graph, _) in enumerate(graphs):
            with torch.cuda.stream(streams[i % 2]):
                graph.replay()
        torch.cuda.synchronize()
        for (_, (o, l)), (_, _, want) in zip(graphs, cases):
            assert torch.equal(o, want[0]) and torch.equal(l, want[1])
            o.zero_()
            l.zero_()
        torch.cuda.synchronize()


def test_page_from_prefill_to_sealed_steps(dev):
    """The operators together: image positions through the rotary update into
    bf16 caches, the prefix sealed, a step's rows appended behind it, attention
    over both, rows dropped by the framework's compaction, and back."""
    from hsd_b200.compaction import compact_kv, keep_indices, plane_pointers
    from hsd_b200.kv8 import Kv8Cache, verify_attention_kv8
    from hsd_b200.plan import SEG_CAUSAL, PackedMask, pack_bits
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    hq, hkv, layers, prefix, sealed = 6, 2, 2, 200, 192
    lens = [5, 1, 30]
    step = sum(lens)
    kv_len = prefix + step
    g = torch.Generator(device=dev).manual_seed(0)
    rot = RotaryAxes([16, 24, 24], device=dev)
    caches = [torch.zeros(1, hkv, kv_len + 10, 128, dtype=torch.bfloat16, device=dev)
              for _ in range(2 * layers)]
    planes = plane_pointers(caches)
    kv8 = Kv8Cache(layers, hkv, 256, device=dev)
    seen = np.arange(kv_len) < prefix
    segs, at = [], 0
    for n in lens:
        segs.append(dict(q_start=at, q_len=n, kind=SEG_CAUSAL, kv=seen))
        at += n
    plan = PackedMask(step, kv_len, segs, device=dev).plan()
    allowed = segments(lens, prefix).to(dev)
    rows = [torch.randn(prefix + step, (hq + 2 * hkv) * 128, generator=g, device=dev)
            .to(torch.bfloat16) for _ in range(layers)]
    pos = torch.randint(0, 60, (3, prefix + step), generator=g, device=dev)
    queries = []
    for l in range(layers):
        for lo, hi in ((0, prefix), (prefix, kv_len)):
            x = rows[l][lo:hi]
            q = rope_append_axes(x[:, :hq * 128], x[:, hq * 128:(hq + hkv) * 128],
                                 x[:, (hq + hkv) * 128:], pos[:, lo:hi], rot, caches[2 * l],
                                 caches[2 * l + 1], lo)
        queries.append(q)
    kv8.seal(planes, sealed)
    kv8.raise_on_device_error()
    bf16 = [c[0].clone() for c in caches]
    for l in range(layers):
        tail = torch.stack([bf16[2 * l], bf16[2 * l + 1]])
        data, scale = kv8.data[l], kv8.scale[l]
        got = verify_attention_kv8(queries[l], kv8.layer(l), kv8.sealed, caches[2 * l],
                                   caches[2 * l + 1], plan)
        check(got, exact(queries[l][0], data, scale, tail, sealed, allowed))
        # near the bf16 cache's attention: sealing moved K and V by half a step
        full = exact(queries[l][0], data, scale, tail, 0, allowed)
        assert (got[0].double() - full[0]).pow(2).mean().sqrt() < 0.05 * full[0].pow(2).mean().sqrt()
    # drop some of the step's rows; the sealed prefix stays where it is
    keep = np.ones(kv_len, bool)
    keep[prefix + 3:prefix + 9] = False
    keep_bits = torch.from_numpy(pack_bits(keep).view(np.int64)).to(dev)[None]
    _, idx, counts = keep_indices(keep_bits, None, kv_len)
    compact_kv(planes, 256, idx, counts=counts)
    torch.cuda.synchronize()
    assert int(counts[0]) == kv_len - 6
    kept = torch.from_numpy(np.nonzero(keep)[0]).to(dev)
    for c, b in zip(caches, bf16):
        assert torch.equal(c[0, :, :kv_len - 6], b[:, kept])
    left = kv_len - 6
    q1 = queries[0][:, :, -1:]
    one = torch.ones(1, left, dtype=torch.bool, device=dev)
    got = verify_attention_kv8(q1, kv8.layer(0), kv8.sealed, caches[0][:, :, :left],
                               caches[1][:, :, :left], plan_of(one))
    check(got, exact(q1[0], kv8.data[0], kv8.scale[0], torch.stack([caches[0][0], caches[1][0]]),
                     sealed, one))
    # sealed rows back in bf16, within half a step of what was sealed
    kv8.unseal(planes, 0, sealed)
    torch.cuda.synchronize()
    for i, (c, b) in enumerate(zip(caches, bf16)):
        s = kv8.scale[i // 2, i % 2, :, :sealed // 64].repeat_interleave(64, -1)[..., None]
        err = (c[0, :, :sealed].float() - b[:, :sealed].float()).abs()
        assert bool((err <= s * 0.5 * (1 + 1e-5) + 2.0 ** -8 * b[:, :sealed].float().abs()).all())
