"""The table of norm_rotary against frequencies of 80 digits; no GPU."""
import decimal

import pytest

import matchattention_b200 as ma

PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")


@pytest.mark.parametrize("theta,rot,axes", [(10000.0, 128, 1), (10000.0, 64, 2), (500000.0, 32, 1), (1.0, 4, 1), (0.001, 32, 1), (1e-6, 256, 2), (1e30, 64, 1)])
def test_entries_are_right_to_half_a_unit(theta, rot, axes):
    table = ma.rotary_frequencies(rot, theta=theta, axes=axes)
    n = rot // 2 // axes
    with decimal.localcontext() as context:
        context.prec = 80
        for j in range(n):
            want = decimal.Decimal(theta) ** (decimal.Decimal(-j) / n) / (2 * PI) * 2 ** 64
            for row in table.tolist():
                assert -2 ** 63 <= row[j] < 2 ** 63
                off = (row[j] - want) % 2 ** 64
                assert min(off, 2 ** 64 - off) <= decimal.Decimal("0.5000001")


def test_extreme_thetas():
    for theta in (5e-324, 1e-300, 1e300):
        assert ma.rotary_frequencies(8, theta=theta).shape == (1, 4)
