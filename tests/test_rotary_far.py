"""Far positions (apply_rotary): an angle is off by no more than the documented
|position| * (inv_freq / 2 pi * 2^-52 + 2^-65) + 2^-26 of a turn, against angles reduced with 60 digits of pi."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def _angle(position, f):
    """position * f modulo 2 pi, f the 64-bit number itself."""
    getcontext().prec = 60
    turn = 2 * PI
    a = Decimal(position) * Decimal(f)
    return float(a - (a / turn).to_integral_value(rounding="ROUND_FLOOR") * turn)


@pytest.mark.gpu
@pytest.mark.parametrize("position", [0, 1, 131071, 2 ** 24 + 1, 2 ** 30 + 12345, 2 ** 31 + 7, 2 ** 40 + 99, -1, -5000, -(2 ** 33) - 3])
def test_far_positions_are_off_by_what_is_documented(position):
    import flash_tree_attn_b200 as fta

    D = 64
    f, _ = fta.rotary_frequencies(D, base=500000.0, scaling="bands", factor=8.0)
    x = torch.zeros(1, 2, 1, D, device="cuda").half()
    x[0, 0, 0, : D // 2] = 1.0      # gives the cosines, then the sines
    x[0, 1, 0, D // 2:] = 1.0       # minus the sines, then the cosines
    y, _ = fta.apply_rotary(x, None, torch.tensor([position], device="cuda"), f)
    y = y[0, :, 0].double().cpu()
    for j, v in enumerate(f.tolist()):
        a = _angle(position, v)
        c, s = math.cos(a), math.sin(a)
        off = abs(position) * (v / (2 * math.pi) * 2.0 ** -52 + 2.0 ** -65) + 2.0 ** -26
        for got, want in ((y[0, j], c), (y[0, D // 2 + j], s), (y[1, j], -s), (y[1, D // 2 + j], c)):
            # the angle, the cosine in 32 bits, the result's rounding to fp16 (half a step, or 2^-25 below its normals)
            assert abs(float(got) - want) <= 2 * math.pi * off + 2.0 ** -22 + max(2.0 ** -11 * abs(want), 2.0 ** -25), (j, float(got), want)
