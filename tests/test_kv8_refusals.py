"""Refusals of the 8-bit cache and the several-axes rotary embedding, and
their oracles against plain arithmetic.  Everything here is rejected on the
host (or never launches): no GPU needed."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from hsd_b200 import _native as N
from oracle import kv8 as OK
from oracle import rope_axes as OA

A = C.c_void_p(256)


def test_rope_axes_c_checks():
    lib = N.load()

    def call(q=A, q_stride=1536, out=A, k=A, k_stride=256, pos=A, axes=3, turns=A, rows=4, hq=12,
             hkv=2, d=128, cache_stride=128, row0=0, head_stride=4096):
        return lib.hsd_rope_append_axes(q, q_stride, out, 1536, k, k_stride, A, 256, pos, 4, 1, axes,
                                        turns, A, 1.0, rows, hq, hkv, d, A, head_stride, A, 4096,
                                        cache_stride, row0, None, None)

    assert call(rows=0) == 0
    assert call(d=64) == 2 and b"head_dim" in lib.hsd_last_error()
    assert call(axes=0) == 2 and call(axes=9) == 2
    for bad in (dict(q=None), dict(out=C.c_void_p(264)), dict(k=C.c_void_p(258)), dict(pos=None),
                dict(pos=C.c_void_p(260)), dict(turns=None), dict(q_stride=1528),
                dict(q_stride=1540), dict(k_stride=248), dict(rows=-1), dict(hkv=0), dict(row0=-1),
                dict(cache_stride=120), dict(head_stride=4097), dict(hq=5000, q_stride=640000)):
        assert call(**bad) == 1, bad
        assert b"bad arguments" in lib.hsd_last_error()


def test_kv8_seal_c_checks():
    lib = N.load()

    def seal(planes=A, n=4, row0=0, data=A, stride=64 * 128, scale=A, sstride=1, b0=0, nb=1):
        return lib.hsd_kv8_seal(planes, n, row0, data, stride, scale, sstride, b0, nb, None, None)

    assert seal(n=0) == 0 and seal(nb=0) == 0
    for bad in (dict(planes=None), dict(data=None), dict(scale=None), dict(n=-1), dict(row0=-1),
                dict(b0=-1), dict(nb=-1), dict(data=C.c_void_p(8)), dict(stride=64 * 128 - 16),
                dict(stride=64 * 128 + 8), dict(sstride=0), dict(b0=1)):
        assert seal(**bad) == 1, bad
    assert seal(n=70000) == 4

    def unseal(row0=0, rows=64, dst=0, planes=A, n=4):
        return lib.hsd_kv8_unseal(A, 64 * 128, A, 1, n, row0, rows, planes, dst, None)

    assert unseal(rows=0) == 0 and unseal(n=0) == 0
    for bad in (dict(row0=-1), dict(rows=-1), dict(dst=-1), dict(row0=1), dict(planes=None)):
        assert unseal(**bad) == 1, bad


def test_verify_attention_kv8_c_checks():
    lib = N.load()
    plan = N.Plan()
    plan.q_len, plan.kv_len = 64, 300

    def call(q=A, q_row=1536, q_head=128, k8=A, h8=256 * 128, ks=A, sh=4, sealed=256, kt=A,
             kt_row=128, kt_head=300 * 128, row0=0, out=A, lse=A, q_len=64, kv_len=300, hq=12, hkv=2,
             d=128, scale=0.1, pl=C.byref(plan), ws=A, ws_bytes=0):
        # ws_bytes = 0: what passes every other check is refused for its workspace
        return lib.hsd_verify_attention_kv8(q, q_row, q_head, k8, h8, k8, h8, ks, ks, sh, sealed, kt,
                                            kt_row, kt_head, kt, kt_row, kt_head, row0, out, lse,
                                            q_len, kv_len, hq, hkv, d, scale, pl, ws, ws_bytes, None,
                                            None)

    def refused(word, code=1, **kw):
        assert call(**kw) == code, kw
        assert word in lib.hsd_last_error(), (kw, lib.hsd_last_error())

    need = lib.hsd_kv8_attention_workspace_bytes(64, 300, 12, 2)
    assert need >= 256
    refused(b"workspace")
    refused(b"workspace", ws=None, ws_bytes=need)
    refused(b"workspace", ws=C.c_void_p(128), ws_bytes=need)
    refused(b"workspace", ws_bytes=need - 1)
    refused(b"workspace", lse=None)
    refused(b"workspace", row0=256, kt_head=44 * 128)
    refused(b"workspace", sealed=0, k8=None, ks=None, h8=0, sh=0)
    refused(b"head_dim", code=2, d=64)
    for scale in (0.0, -0.1, math.nan, math.inf):
        refused(b"scale", scale=scale)
    for bad in (dict(pl=None), dict(q_len=65), dict(kv_len=299), dict(hq=0), dict(hkv=0), dict(hq=13),
                dict(q=None), dict(q=C.c_void_p(8)), dict(q_row=1540), dict(q_head=0), dict(out=None),
                dict(out=C.c_void_p(264)), dict(lse=C.c_void_p(258)), dict(sealed=-64),
                dict(sealed=100), dict(sealed=320), dict(row0=-1), dict(row0=257), dict(k8=None),
                dict(k8=C.c_void_p(264)), dict(ks=None), dict(ks=C.c_void_p(258)),
                dict(h8=256 * 128 - 16), dict(h8=256 * 128 + 8), dict(sh=3), dict(kt=None),
                dict(kt_row=132), dict(kt_head=0)):
        refused(b"bad arguments", **bad)
    for bad in ((0, 300, 12, 2), (64, 0, 12, 2), (64, 300, 0, 2), (64, 300, 12, 0), (64, 300, 12, 5)):
        assert lib.hsd_kv8_attention_workspace_bytes(*bad) == 0


def test_rotary_axes_refusals_and_tables():
    from hsd_b200.rope import RotaryAxes
    for bad in (dict(sections=[]), dict(sections=[32, 31]), dict(sections=[-1, 65]),
                dict(sections=[1] * 64), dict(sections=[16, 24, 24], interleaved=True),
                dict(sections=[64], theta=0.0), dict(sections=[64], inv_freq=[1.0] * 63),
                dict(sections=[64], inv_freq=[math.nan] * 64),
                dict(sections=[64], scaling=math.inf)):
        with pytest.raises(ValueError):
            RotaryAxes(device="cpu", **bad)
    for sections, inter in (([16, 24, 24], False), ([24, 20, 20], True), ([0, 64], False)):
        r = RotaryAxes(sections, interleaved=inter, device="cpu")
        assert r.pair_axis.tolist() == OA.pair_axis(sections, inter) and r.axes == len(sections)
    # the fixed-point turns against long double: within half a unit of 2^-64, as far as that shows
    r = RotaryAxes([64], theta=1e4, device="cpu")
    t = (r.turns.numpy().view(np.uint64).astype(np.longdouble)) / np.longdouble(2) ** 64
    want = np.array([np.longdouble(1e4 ** (-i / 64)) for i in range(64)]) \
        / (2 * np.longdouble("3.14159265358979323846264338327950288"))
    assert np.abs(t - want).max() < 2.0 ** -62
    # a turn more per position is no turn
    two_pi = 2 * math.pi
    a = RotaryAxes([64], inv_freq=[0.25] * 64, device="cpu").turns
    b = RotaryAxes([64], inv_freq=[0.25 + two_pi] * 64, device="cpu").turns
    assert (a - b).abs().max().item() < 2 ** 64 * 1e-15


def test_rope_append_axes_refusals():
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    kc = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(TypeError):  # host tensors
        rope_append_axes(x, x, x, torch.zeros(1, 4, dtype=torch.int64),
                         RotaryAxes([64], device="cpu"), kc, kc, 0)


def test_kv8_cache_refusals():
    from hsd_b200.kv8 import Kv8Cache
    for bad in ((0, 2, 64), (1, 0, 64), (1, 1, 0), (1, 1, 100)):
        with pytest.raises(ValueError):
            Kv8Cache(*bad, device="cpu")
    c = Kv8Cache(2, 2, 256, device="cpu")
    planes = torch.zeros(8, dtype=torch.int64)
    for bad in (63, -64, 320):
        with pytest.raises(ValueError):
            c.seal(planes, bad)
    with pytest.raises(ValueError):
        c.seal(planes[:7], 64)
    with pytest.raises(ValueError):
        c.seal(planes.int(), 64)
    with pytest.raises(ValueError):
        c.seal(planes, 64, src_row0=-1)
    with pytest.raises(ValueError):
        c.unseal(planes, 0, 1)      # nothing sealed yet
    with pytest.raises(ValueError):
        c.reset(64)
    k, v, ks, vs = c.layer(1)
    assert k.shape == v.shape == (2, 256, 128) and ks.shape == vs.shape == (2, 4)


def test_seal_oracle_against_fractions():
    from fractions import Fraction as F
    rng = np.random.default_rng(0)
    x = torch.from_numpy(rng.standard_normal((1, 64, 128)) * 3).to(torch.bfloat16)
    n, s = OK.seal(x)
    amax = max(abs(F(float(t))) for t in x.flatten()[:].tolist())
    for i, t in enumerate(x.flatten().tolist()[:2000]):
        assert int(n.flatten()[i]) == round(127 * F(t) / amax)
    assert abs(s[0, 0] - float(amax) / 127) <= 1e-16 * float(amax)
    # each value is within half a step of the value it is held as
    err = np.abs(OK.values(n, s) - x.double().numpy())
    assert (err <= s[0, 0] * (0.5 + 127 * 2.0 ** -24)).all()


def test_rope_axes_oracle_is_a_rotation():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 3, 128))
    pos = rng.integers(-1000, 1000, (2, 5))
    freq = [1e6 ** (-i / 64) for i in range(64)]
    axis = OA.pair_axis([40, 24])
    y = OA.rotate(x, pos, axis, freq)
    assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))
    assert np.allclose(OA.rotate(y, -pos, axis, freq), x)
