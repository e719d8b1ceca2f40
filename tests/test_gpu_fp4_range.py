"""The fp4 product over the range of bfloat16: factors whose product fits although a product on the way might not."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    import duqlinear4bitcuda_b200._CUDA as o
    return o


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("m,n,k", [(3, 200, 512), (200, 520, 1056)])
@pytest.mark.parametrize("power", [118, 112, 60, -60, -96])
def test_tokens_scaled_by_a_power_of_two(fmt, m, n, k, power):
    """Codes do not change when a token is scaled by a power of two, its scale does exactly, and so does the result wherever it is
    a normal number. Weights are of about 2^-24, so that results of the largest tokens still fit."""
    g = torch.Generator().manual_seed(m + power)
    x = (torch.randn(m, k, generator=g) * 0.5).bfloat16().cuda()
    w = (torch.randn(n, k, generator=g) * 2.0 ** -24).bfloat16().cuda()
    qw = ops().fp4_quantize(fmt, w)
    want = ops().linear_fp4_from_16bit(fmt, x, *qw)
    assert want.isfinite().all() and want.abs().max() > 0
    scaled = (x.double() * 2.0 ** power).bfloat16()
    got = ops().linear_fp4_from_16bit(fmt, scaled, *qw)
    exact = want.double() * 2.0 ** power
    normal = exact.abs() >= torch.finfo(torch.bfloat16).tiny
    assert normal.float().mean() > 0.9
    assert got.isfinite().all() and torch.equal(got.double()[normal], exact[normal])
