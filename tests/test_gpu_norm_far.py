"""norm_rotary at far positions against angles of 80 digits."""
import decimal
import math

import pytest
import torch

import _dense
from _dense import assert_within

pytestmark = pytest.mark.gpu
PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")


def turns(position, j, n):
    """The fraction of a turn that is left of position * 10000 ** (-j / n) / (2 pi)."""
    with decimal.localcontext() as context:
        context.prec = 80
        return float(position * decimal.Decimal(10000) ** (decimal.Decimal(-j) / n) / (2 * PI) % 1)


@pytest.mark.parametrize("start", [0, 10 ** 6, 2 ** 31, 2 ** 40, -2 ** 40])
def test_far_positions(start):
    """float32: the angle is off by 2^-26 turns, by 2^-65 turns per position for the table, and by what sincospif adds (within the bounds of
    _dense.norm: its 2^-24 pi per term is a part of (d + 16) 2^-22)."""
    import matchattention_b200 as ma
    N, d = 24, 64
    at = [start + 37 * i for i in range(N)]
    q = torch.randn(1, N, 2, d, generator=torch.Generator().manual_seed(61)).cuda()
    angle = 2 * math.pi * torch.tensor([[turns(p, j, d // 2) for j in range(d // 2)] for p in at], dtype=torch.float64, device="cuda")[None, :, None]
    freqs = ma.rotary_frequencies(d, device="cuda")
    got = ma.norm_rotary(q, None, freqs, torch.tensor(at, device="cuda"))
    want, bound = _dense.norm(q, None, freqs, angle, 1e-6)
    far = 2 * math.pi * (2.0 ** -26 + abs(start) * 2.0 ** -65)
    unit = want[0].abs()
    other = torch.cat((unit[..., d // 2:], unit[..., :d // 2]), -1)
    assert_within(got, want[0], bound[0] + far * (unit + other), "q")
