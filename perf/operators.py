"""The operators of the page cache, as cases that can be timed and checked.

Three operators around the KV cache of a packed page (head_dim 128 throughout):

* ``rope``: rotary positions with several axes, with the cache update -- the
  queries rotated, the rotated keys and the values written to their rows of
  the layer's cache;
* ``seal``: whole 64-token blocks of every layer's planes into the 8-bit
  cache (one scale for each block of tokens and head) and back to bf16 rows;
* ``attn``: packed verification attention over a cache whose first ``sealed``
  columns are held in 8 bits and whose other columns are bf16.

``run`` computes them in plain torch operations, or with ``own`` through the
package's entry points.
"""
import math

import torch

own = False

D = 128
BLOCK = 64          # tokens that share a scale
MIN_AMAX = 2.0 ** -100


# ---------------------------------------------------------------- cases
def _rope(name, rows, hq, hkv, sections, far, interleaved=False, theta=1e6):
    """``sections``: dimension pairs of each position axis; ``far``: largest position."""
    return {"name": name, "kind": "rope", "rows": rows, "hq": hq, "hkv": hkv,
            "sections": sections, "far": far, "interleaved": interleaved, "theta": theta}


def _seal(name, layers, hkv, rows):
    return {"name": name, "kind": "seal", "layers": layers, "hkv": hkv, "rows": rows}


def _attn(name, hq, hkv, sealed, prefix, lens, pad):
    """``prefix`` columns that every segment sees (``sealed`` of them in 8
    bits), then the causal segments ``lens``; ``pad``: rows up to a multiple of
    128 that see nothing."""
    return {"name": name, "kind": "attn", "hq": hq, "hkv": hkv, "sealed": sealed,
            "prefix": prefix, "lens": lens, "pad": pad}


# draft lengths of a region page (median 60) and of a page of short regions (median 40)
_REGIONS = ("61,34,118,47,72,25,90,63,55,140,38,81,60,29,104,66,44,77,52,160,"
            "33,58,95,41,70,62,27,112,49,84,57,36")
_SHORT = ("41,22,77,30,48,17,60,39,36,95,25,54,40,19,69,44,29,51,35,107,22,39,63,27,"
          "47,41,18,75,33,56,38,24,52,31,43,88,20,37,46,28,65,34,42,23,58,32,49,26")


def listed():
    return [
        # one new token of a page that is read to its end: 4 axes, 16/8 heads
        _rope("rope_token", 1, 16, 8, "16,16,16,16", 4096),
        # the packed rows of a region page's step, 12/2 heads, time / height / width
        _rope("rope_regions", 2176, 12, 2, "16,24,24", 6000),
        # several pages' prompts at once, axes interleaved over the pairs
        _rope("rope_prompts", 16640, 16, 8, "24,20,20", 120000, interleaved=True),
        # the block that has just filled, every layer of a small decoder
        _seal("seal_block", 24, 8, 64),
        # a page's image prefix, 28 layers with 2 KV heads
        _seal("seal_page", 28, 2, 2560),
        # several pages' prefixes in one row range
        _seal("seal_pages", 28, 2, 8000),
        # the last block of a page decodes token by token
        _attn("attn_token", 12, 2, 2560, 2624, "1", False),
        # the same, far into a long document
        _attn("attn_long_token", 16, 8, 131008, 131050, "1", False),
        # forty regions, one row each (no draft matched)
        _attn("attn_single_rows", 12, 2, 2560, 2624, ",".join(["1"] * 40), False),
        # a region page's verification step
        _attn("attn_regions", 12, 2, 2560, 2624, _REGIONS, True),
        # many short regions, 16/8 heads
        _attn("attn_short_regions", 16, 8, 1600, 1600, _SHORT, True),
        # one page draft over several pages of context
        _attn("attn_page", 12, 2, 16384, 16401, "2049", False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = ((12, 2), (16, 8), (8, 1), (4, 4), (28, 4), (6, 2), (5, 1), (32, 8))


def draw(rng):
    kind = rng.choice(("rope", "seal", "attn", "attn"))
    hq, hkv = rng.choice(_HEADS)
    if kind == "rope":
        axes = rng.randint(1, 4)
        cuts = sorted(rng.sample(range(1, 64), axes - 1))
        sec = [b - a for a, b in zip([0] + cuts, cuts + [64])]
        interleaved = rng.random() < 0.4
        if interleaved:  # an equal share for the later axes, the rest to the first
            s = rng.randint(1, 64 // axes)
            sec = [64 - s * (axes - 1)] + [s] * (axes - 1)
        c = _rope("", _log(rng, 1, 530000 // (hq + 2 * hkv)), hq, hkv,
                  ",".join(str(s) for s in sec), _log(rng, 2, 131072), interleaved,
                  rng.choice((1e4, 5e5, 1e6)))
    elif kind == "seal":
        layers = rng.randint(1, 28)
        c = _seal("", layers, hkv, BLOCK * _log(rng, 1, min(128, 14000 // (2 * layers * hkv))))
    else:
        prefix = _log(rng, 64, 131072)
        sealed = rng.choice((prefix, max(0, prefix - rng.randint(0, 500)), prefix // 2)) // BLOCK
        most = max(1, min(2304, int(3.0e8 / (prefix * hq)), int(2.0e6 / (hq * D))))
        total = _log(rng, 1, most)
        shape = rng.choice(("one", "single", "mixed"))
        if shape == "one":
            lens = [total]
        elif shape == "single":
            lens = [1] * min(total, 200)
        else:
            lens, left = [], total
            while left > 0:
                n = min(left, max(1, int(round(rng.lognormvariate(math.log(50), 0.6)))))
                lens.append(n)
                left -= n
        c = _attn("", hq, hkv, sealed * BLOCK, prefix, ",".join(str(n) for n in lens),
                  rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------- shared shapes
def _sections(case):
    return [int(s) for s in case["sections"].split(",")]


def _pair_axis(case):
    """The position axis of each of the 64 dimension pairs."""
    sec = _sections(case)
    if not case["interleaved"]:
        return [a for a, n in enumerate(sec) for _ in range(n)]
    n = len(sec)
    return [i % n if i < n * sec[i % n] else 0 for i in range(64)]


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def _q_len(case):
    n = sum(_lens(case))
    return (n + 127) // 128 * 128 if case["pad"] else n


def _allowed(case, device):
    """bool [Q, KV]: the columns each packed row attends to."""
    q_len, prefix = _q_len(case), case["prefix"]
    a = torch.zeros(q_len, prefix + q_len, dtype=torch.bool, device=device)
    at = 0
    for n in _lens(case):
        a[at:at + n, :prefix] = True
        a[at:at + n, prefix + at:prefix + at + n] = torch.ones(
            n, n, dtype=torch.bool, device=device).tril()
        at += n
    return a


# ---------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _prepare_rope(case, g):
    rows, hq, hkv = case["rows"], case["hq"], case["hkv"]
    axes = len(_sections(case))
    qkv = (_normal(g, rows, (hq + 2 * hkv) * D) * 2).to(torch.bfloat16)
    pos = torch.randint(0, case["far"], (axes, rows), generator=g, device="cuda")
    row0 = 37
    cap = row0 + rows + 5
    s = {"kind": "rope", "case": case, "qkv": qkv, "pos": pos, "row0": row0,
         "q_out": torch.zeros(rows, hq * D, dtype=torch.bfloat16, device="cuda"),
         "k_cache": _normal(g, hkv, cap, D).to(torch.bfloat16),
         "v_cache": _normal(g, hkv, cap, D).to(torch.bfloat16)}
    if own:
        from hsd_b200.rope import RotaryAxes
        s["rotary"] = RotaryAxes(_sections(case), theta=case["theta"],
                                 interleaved=case["interleaved"], device="cuda")
    else:
        s["axis"] = torch.tensor(_pair_axis(case), device="cuda")
        s["inv_freq"] = torch.tensor([case["theta"] ** (-2 * i / D) for i in range(D // 2)],
                                     dtype=torch.float64, device="cuda")
    return s


def _prepare_seal(case, g):
    layers, hkv, rows = case["layers"], case["hkv"], case["rows"]
    # heads and channels of unlike magnitude, as keys have
    mag = torch.exp(_normal(g, layers, 2, hkv, 1, D) * 0.8)
    cache = (_normal(g, layers, 2, hkv, rows, D) * mag).to(torch.bfloat16)
    s = {"kind": "seal", "case": case, "cache": cache, "back": torch.empty_like(cache)}
    if own:
        from hsd_b200.compaction import plane_pointers
        from hsd_b200.kv8 import Kv8Cache
        s["kv8"] = Kv8Cache(layers, hkv, rows, device="cuda")
        s["planes"] = plane_pointers(list(cache.flatten(0, 1)))
        s["back_planes"] = plane_pointers(list(s["back"].flatten(0, 1)))
    return s


def _prepare_attn(case, g):
    hq, hkv, sealed = case["hq"], case["hkv"], case["sealed"]
    q_len = _q_len(case)
    kv_len = case["prefix"] + q_len
    q = _normal(g, hq, q_len, D)
    # some rows attend to few columns, most to many
    q = q * torch.where(torch.rand(hq, q_len, 1, generator=g, device="cuda") < 0.2, 4.0, 1.0)
    nb = max(sealed // BLOCK, 1)
    mag = torch.exp(_normal(g, 2, hkv, nb, 1) * 0.2)
    x = _normal(g, 2, hkv, nb, BLOCK * D)
    amax = x.abs().amax(-1, keepdim=True)
    data = torch.round(x * (127 / amax)).to(torch.int8).view(2, hkv, nb * BLOCK, D)
    scale = (amax * mag / 127).view(2, hkv, nb)
    tail = _normal(g, 2, hkv, kv_len - sealed, D).to(torch.bfloat16)
    s = {"kind": "attn", "case": case, "q": q.to(torch.bfloat16), "data": data, "scale": scale,
         "tail": tail, "sm_scale": 1 / math.sqrt(D)}
    if own:
        import numpy as np

        from hsd_b200.kv8 import Kv8Layer
        from hsd_b200.plan import SEG_CAUSAL, PackedMask
        seen = np.arange(kv_len) < case["prefix"]
        segs, at = [], 0
        for n in _lens(case):
            segs.append(dict(q_start=at, q_len=n, kind=SEG_CAUSAL, kv=seen))
            at += n
        s["plan"] = PackedMask(q_len, kv_len, segs, device="cuda").plan()
        s["layer"] = Kv8Layer(data[0], data[1], scale[0], scale[1])
    else:
        s["allowed"] = _allowed(case, "cuda")
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"rope": _prepare_rope, "seal": _prepare_seal, "attn": _prepare_attn}[case["kind"]](
        case, g)


# ---------------------------------------------------------------- one pass
def _rope_own(s):
    from hsd_b200.rope import rope_append_axes
    c = s["case"]
    a, b = c["hq"] * D, (c["hq"] + c["hkv"]) * D
    q = rope_append_axes(s["qkv"][:, :a], s["qkv"][:, a:b], s["qkv"][:, b:], s["pos"],
                         s["rotary"], s["k_cache"], s["v_cache"], s["row0"], out=s["q_out"])
    return q, s["k_cache"], s["v_cache"]


def _rotate(x, cos, sin):
    """x [rows, heads, 128], cos / sin [rows, 64] -> [heads, rows, 128] bf16"""
    x = x.float()
    lo, hi = x[..., :64], x[..., 64:]
    cos, sin = cos[:, None], sin[:, None]
    y = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    return y.to(torch.bfloat16).transpose(0, 1)


def _rope_plain(s):
    c = s["case"]
    rows, hq, hkv = c["rows"], c["hq"], c["hkv"]
    # 64 bits: positions of far tokens times a frequency
    ang = s["pos"][s["axis"]].t().double() * s["inv_freq"]
    cos, sin = ang.cos().float(), ang.sin().float()
    x = s["qkv"].view(rows, hq + 2 * hkv, D)
    at = slice(s["row0"], s["row0"] + rows)
    q = _rotate(x[:, :hq], cos, sin)
    s["k_cache"][:, at] = _rotate(x[:, hq:hq + hkv], cos, sin)
    s["v_cache"][:, at] = x[:, hq + hkv:].transpose(0, 1)
    return q[None], s["k_cache"], s["v_cache"]


def _seal_own(s):
    kv8, rows = s["kv8"], s["case"]["rows"]
    kv8.reset()
    kv8.seal(s["planes"], rows, src_row0=0)
    kv8.unseal(s["back_planes"], 0, rows, dst_row0=0)
    return s["back"], kv8.scale


def _seal_plain(s):
    c = s["case"]
    # 64 bits: values on the border between two steps go to the even one
    x = s["cache"].double().view(c["layers"], 2, c["hkv"], c["rows"] // BLOCK, BLOCK * D)
    amax = x.abs().amax(-1).clamp_min(MIN_AMAX)
    n = torch.round(x * 127 / amax[..., None])
    scale = (amax / 127).float()
    s["back"].copy_((n.float() * scale[..., None]).view_as(s["cache"]))
    return s["back"], scale


def _attn_own(s):
    from hsd_b200.kv8 import verify_attention_kv8
    sealed = s["case"]["sealed"]
    return verify_attention_kv8(s["q"], s["layer"], sealed, s["tail"][0], s["tail"][1], s["plan"],
                                scale=s["sm_scale"], tail_row0=sealed)


def _attn_plain(s):
    c = s["case"]
    hq, hkv, sealed = c["hq"], c["hkv"], c["sealed"]
    allowed = s["allowed"]
    nb = sealed // BLOCK
    group = hq // hkv
    out = torch.empty(allowed.shape[0], hq, D, dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(hq, allowed.shape[0], dtype=torch.float32, device="cuda")
    for h in range(hkv):
        k, v = (torch.cat([(s["data"][i, h, :sealed].float().view(nb, BLOCK * D)
                            * s["scale"][i, h, :nb, None]).view(sealed, D),
                           s["tail"][i, h].float()]) for i in (0, 1))
        for a in range(h * group, (h + 1) * group):
            x = (s["q"][a].float() @ k.t()) * s["sm_scale"]
            x = x.masked_fill(~allowed, -math.inf)
            m = x.amax(-1, keepdim=True)
            m = torch.where(torch.isinf(m), 0.0, m)
            p = torch.exp(x - m)
            total = p.sum(-1, keepdim=True)
            o = (p @ v) / torch.where(total > 0, total, 1.0)
            out[:, a] = o.to(torch.bfloat16)
            lse[a] = (m + torch.log(total))[:, 0]
    return out, lse


def run(state):
    """One pass; rope: (rotated queries [1, Hq, rows, 128], k_cache, v_cache),
    seal: (the sealed rows' values, scales), attn: (out [Q, Hq, 128], lse)."""
    k = state["kind"]
    if own:
        return {"rope": _rope_own, "seal": _seal_own, "attn": _attn_own}[k](state)
    return {"rope": _rope_plain, "seal": _seal_plain, "attn": _attn_plain}[k](state)


# ---------------------------------------------------------------- work
def work(case):
    if case["kind"] == "rope":
        heads = case["hq"] + 2 * case["hkv"]
        return {"bytes": case["rows"] * (heads * D * 4 + 8 * len(_sections(case))),
                "flops": case["rows"] * (case["hq"] + case["hkv"]) * D * 3}
    if case["kind"] == "seal":
        n = case["layers"] * 2 * case["hkv"] * case["rows"] * D
        # rows read, 8-bit values written and read back, rows written, scales twice
        return {"bytes": n * 6 + n // (BLOCK * D) * 8, "flops": n * 4}
    hq, hkv, prefix, sealed = case["hq"], case["hkv"], case["prefix"], case["sealed"]
    q_len, lens = _q_len(case), _lens(case)
    pairs = sum(n * prefix + n * (n + 1) // 2 for n in lens)
    kv = 2 * hkv * (sealed * D + sealed // BLOCK * 4 + (prefix - sealed + sum(lens)) * D * 2)
    return {"bytes": kv + q_len * hq * (D * 4 + 4), "flops": 4 * D * hq * pairs}


# ---------------------------------------------------------------- 64 bits
def _exact_rope(s):
    c = s["case"]
    rows, hq, hkv = c["rows"], c["hq"], c["hkv"]
    pos = s["pos"].double()
    x = s["qkv"].double().view(rows, hq + 2 * hkv, D)
    y = x.clone()
    for i, axis in enumerate(_pair_axis(c)):
        ang = pos[axis] * math.pow(c["theta"], -i / 64)
        co, si = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        n = hq + hkv
        y[:, :n, i] = x[:, :n, i] * co - x[:, :n, i + 64] * si
        y[:, :n, i + 64] = x[:, :n, i + 64] * co + x[:, :n, i] * si
    y = y.permute(1, 0, 2)
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    kc[:, s["row0"]:s["row0"] + rows] = y[hq:hq + hkv]
    vc[:, s["row0"]:s["row0"] + rows] = y[hq + hkv:]
    return y[None, :hq], kc, vc


def _exact_seal(s):
    c = s["case"]
    back = torch.empty(s["cache"].shape, dtype=torch.float64, device="cuda")
    scale = torch.empty(c["layers"], 2, c["hkv"], c["rows"] // BLOCK, dtype=torch.float64,
                        device="cuda")
    for b in range(c["rows"] // BLOCK):
        x = s["cache"][:, :, :, b * BLOCK:(b + 1) * BLOCK].double()
        top = x.abs().amax((-1, -2)).clamp_min(MIN_AMAX)
        # 127 x is exact (bf16 values), so one division decides the border values
        n = torch.round(127 * x / top[..., None, None])
        scale[..., b] = top / 127
        back[:, :, :, b * BLOCK:(b + 1) * BLOCK] = n * scale[..., b][..., None, None]
    return back, scale


def _exact_attn(s):
    c = s["case"]
    hq, group, sealed, prefix = c["hq"], c["hq"] // c["hkv"], c["sealed"], c["prefix"]
    q_len = _q_len(c)
    out = torch.zeros(q_len, hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((hq, q_len), -math.inf, dtype=torch.float64, device="cuda")
    kv = torch.cat([s["data"][:, :, :sealed].double()
                    * s["scale"][:, :, :sealed // BLOCK].double().repeat_interleave(
                        BLOCK, -1)[..., None], s["tail"].double()], 2)
    for a in range(hq):
        k, v = kv[0, a // group], kv[1, a // group]
        at = 0
        for n in _lens(c):
            rows = s["q"][a, at:at + n].double()
            kk = torch.cat([k[:prefix], k[prefix + at:prefix + at + n]])
            vv = torch.cat([v[:prefix], v[prefix + at:prefix + at + n]])
            x = (rows @ kk.t()) * s["sm_scale"]
            i = torch.arange(n, device="cuda")
            x[:, prefix:] = torch.where(i[None] <= i[:, None], x[:, prefix:], -math.inf)
            lse[a, at:at + n] = torch.logsumexp(x, -1)
            out[at:at + n, a] = torch.softmax(x, -1) @ vv
            at += n
    return out, lse


def exact(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = case["kind"]
    if k == "rope":
        return _exact_rope(_prepare_rope(case, g))
    if k == "seal":
        return _exact_seal(_prepare_seal(case, g))
    return _exact_attn(_prepare_attn(case, g))
