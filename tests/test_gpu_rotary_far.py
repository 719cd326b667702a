"""Rotary tables at far positions against angles in 60 decimal digits.  A pair's frequency is held in 2^-64 of a turn,
with the roundings of up to 255 products of 64 significant bits: at most 2^-57 of a turn off, and 2^-61 from a theta of
10^4 on, where the frequencies fall faster than the roundings add up.  A position multiplies that; what a near position
may be off by (a fraction of a turn brought to fp32, its two sums and their roundings: 2^-21) comes on top."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

pytestmark = pytest.mark.gpu
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")


def _reference(positions, dim, theta):
    getcontext().prec = 60
    turns = [Decimal(theta) ** (Decimal(-2 * i) / Decimal(dim)) / (2 * PI) for i in range(dim // 2)]
    out = []
    for p in positions:
        angles = [float((Decimal(p) * t) % 1) * 2 * math.pi for t in turns]
        out.append([[math.cos(a), math.sin(a)] for a in angles])
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("theta", [1.5, 100.0, 1e4, 1e6])
@pytest.mark.parametrize("dim", [8, 56, 128, 512])
@pytest.mark.parametrize("dtype", [torch.int64, torch.float32])
def test_far_positions(theta, dim, dtype):
    import qlin
    pos = [0, 1, 32760, 2 ** 24 - 1, 2 ** 28, 2 ** 32, 2 ** 40, -(2 ** 40), 2 ** 45]
    if dtype == torch.int64:
        pos += [2 ** 28 + 1, 2 ** 32 - 1, -(2 ** 33) + 5, 2 ** 40 + 1, 2 ** 45 - 3]
    else:
        pos += [0.1875, -17.0625, 2.0 ** -30, 3 * 2.0 ** 40]
    got = qlin.rotary_table(torch.tensor(pos, dtype=dtype, device="cuda").unsqueeze(1), [dim], theta).double().cpu()
    off = (got - _reference(pos, dim, theta)).abs().amax((1, 2))
    unit = 2.0 ** (-61 if theta >= 1e4 else -57)
    for p, e in zip(pos, off.tolist()):
        assert e <= 2.0 ** -21 + 2 * math.pi * abs(p) * unit, (p, e)
