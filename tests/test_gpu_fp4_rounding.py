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


def _product(silu, up):
    return (silu.float() * up.float()).to(silu.dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("pin", [16.0, 128.0])
def test_silu_of_every_gate(dtype, pin):
    """Each finite gate whose silu is not too small, twice, with the ups between which its product passes 2.5, the border of the
    codes of 2 and 3 under a scale of 1. The first of each block of 32 pins that scale with a product of 4 (and, by its own gate,
    which of the two quotients its neighbour takes). A silu that is one unit off would show in most of these codes."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).cuda()
    g = bits.view(dtype)
    s = torch.nn.functional.silu(g)
    big = torch.finfo(dtype).max / 2        # ups stay finite; bfloat16's also stay normal
    keep = g.isfinite() & (s.abs() > 2.5 / big) & (s.abs() < big)
    g, s = g[keep], s[keep]
    assert g.numel() > 20000
    # the first up (by magnitude) whose product is beyond 2.5: from a few units below the quotient upwards
    near = (2.5 / s.double()).to(dtype).view(torch.int16)
    ups = torch.stack([(near + d).view(dtype) for d in range(-4, 5)])
    beyond = _product(s, ups).abs() > 2.5
    assert beyond[-1].all() and not beyond[0].any()
    first = beyond.int().argmax(0, keepdim=True)
    hi, lo = ups.gather(0, first)[0], ups.gather(0, first - 1)[0]

    def blocks(t, pinned):
        t = torch.cat([t, t[-1:].expand(-t.numel() % (31 * 8))]).view(-1, 31)
        return torch.cat([torch.full_like(t[:, :1], pinned), t], 1).view(-1, 256)
    gate, up = blocks(torch.cat([g, g]), pin), blocks(torch.cat([hi, lo]), 4 / pin)
    silu = blocks(torch.cat([s, s]), pin)
    want = ops().fp4_quantize("mxfp4", _product(silu, up))[0]
    assert torch.equal(ops().fp4_silu_mul_quantize("mxfp4", torch.cat([gate, up], 1))[0], want)
    for d in (-1, 1):   # the cases tell a silu apart that is one unit smaller or larger
        off = blocks((torch.cat([s, s]).view(torch.int16) + d).view(dtype), pin)
        other = ops().fp4_quantize("mxfp4", _product(off, up))[0]
        assert (other != want).sum() > g.numel() // 4
