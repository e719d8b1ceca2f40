"""Roundings of the norm joint and of the SiLU product at the places where an error of a few units shows."""
from fractions import Fraction

import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    import duqlinear4bitcuda_b200._CUDA as o
    return o


def _root(f):
    """1 / f^2 - 1 as the nearest double, for a fraction f: the eps with which a row of ones has the reciprocal root f."""
    return float(1 / (f * f) - 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 300])
def test_reciprocal_root_next_to_a_border(dtype, rows):
    """Rows of ones, whose mean of squares is exactly 1, and an eps that puts 1 / sqrt(1 + eps) a relative 4e-15 beside the middle
    of two floats, of which one rounds to the 16-bit number below and one to that above. eps (rounded to a double), 1 + eps
    and the root's own operations in 64 bits are off by at most a few 2^-53 together, less than 2e-15: the side that the 16-bit
    result lies on is the exact root's."""
    bits = 11 if dtype == torch.float16 else 8
    x = torch.ones(rows, 32, dtype=dtype, device="cuda")
    w = torch.ones(32, dtype=dtype, device="cuda")
    step = Fraction(1, 2 ** bits)                  # of 16-bit numbers in [0.5, 1)
    first = 2 ** (bits - 1)
    wrong = []
    for i in range(0, first - 1, first // 128 | 1):
        below, above = (first + i) * step, (first + i + 1) * step
        tie = below + step / 2
        # floats in [0.5, 1) are 2^-24 apart; the tie itself goes to the even 16-bit number
        middle = tie + Fraction(-1 if (first + i) % 2 else 1, 2 ** 25)
        for side, want in ((-1, below), (1, above)):
            eps = _root(middle * (1 + side * Fraction(4, 10 ** 15)))
            got = ops().norm_residual_quantize("none", x, w, eps)[1]
            if not (got == float(want)).all():
                wrong.append((float(middle), side))
    assert not wrong, (len(wrong), wrong[:4])
