"""Far positions of the several-axes rotary embedding: the table's angle against
exact fractions, and the kernel's against the table's."""
import math
from fractions import Fraction

import pytest
import torch

# 2 pi to 60 digits
TWO_PI = Fraction("6.28318530717958647692528676655900576839433879875021164194988918")
POSITIONS = [1, -7, 4097, 2 ** 31 + 5, -2 ** 39, 2 ** 40 + 3, 2 ** 52 - 1, -2 ** 62 - 12345,
             2 ** 63 - 1, -2 ** 63]


def _freq(theta):
    return [float(theta) ** (-i / 64) for i in range(64)]


def test_table_angle_is_off_by_half_a_unit_per_position():
    from hsd_b200.rope import RotaryAxes
    for theta in (1e4, 1e6):
        turns = RotaryAxes([64], theta=theta, device="cpu").turns.tolist()
        for t, f in zip(turns, _freq(theta)):
            for pos in POSITIONS:
                off = Fraction(t * pos, 2 ** 64) - Fraction(f) * pos / TWO_PI
                off -= round(off)
                assert abs(off) <= abs(pos) * Fraction(1, 2 ** 65) + Fraction(1, 2 ** 100)


@pytest.mark.gpu
def test_kernel_turns_by_the_tables_angle_at_any_position():
    """Angle off by 2^-25 + 2^-31 half turns (below 2^-23 rad), cosine and sine by
    2^-23 more, then half a bf16 step."""
    from hsd_b200.rope import RotaryAxes, rope_append_axes
    dev = torch.device("cuda:0")
    n = len(POSITIONS)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(n, 128, generator=g).to(torch.bfloat16)
    rot = RotaryAxes([64], theta=1e4, device=dev)
    kc = torch.zeros(1, n, 128, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    rope_append_axes(None, x.to(dev), x.to(dev),
                     torch.tensor([POSITIONS], dtype=torch.int64, device=dev), rot, kc, vc, 0)
    got = kc[0].double().cpu()
    turns = rot.turns.cpu().tolist()
    for r, pos in enumerate(POSITIONS):
        for i, t in enumerate(turns):
            m = t * pos % 2 ** 64
            a = 2 * math.pi * ((m - 2 ** 64 if m >= 2 ** 63 else m) / 2 ** 64)
            lo, hi = float(x[r, i]), float(x[r, i + 64])
            for j, want in ((i, lo * math.cos(a) - hi * math.sin(a)),
                            (i + 64, hi * math.cos(a) + lo * math.sin(a))):
                tol = 2.0 ** -8 * abs(want) + 2.0 ** -21 * (abs(lo) + abs(hi))
                assert abs(float(got[r, j]) - want) <= tol, (pos, i)
