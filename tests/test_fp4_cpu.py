"""CPU-only: refusals of the microscaled 4-bit entry points, the order of the block scales, the module's state."""
import ctypes

import numpy as np
import pytest
import torch

from tests import _fp4 as F

H, B = torch.float16, torch.bfloat16
P = 0x1000          # a 16-byte aligned non-NULL address; a call that reached a launch would fail with a positive status


def test_scale_bytes_and_workspace():
    import duqlinear4bitcuda_b200.lib as L
    c = L.cdll
    assert c.duq4_fp4_scale_bytes(L.FP4_MX, 1, 32) == 512
    assert c.duq4_fp4_scale_bytes(L.FP4_NV, 129, 96) == 2 * 2 * 512
    assert c.duq4_fp4_scale_bytes(L.FP4_NV, 28672, 8192) == 28672 * 8192 // 16
    assert c.duq4_fp4_scale_bytes(3, 128, 128) == 0
    assert c.duq4_fp4_scale_bytes(L.FP4_NV, 0xFFFFFFFF, 65536) == 2 ** 25 * 1024 * 512   # beyond 32 bits
    assert c.duq4_linear_fp4_workspace_bytes(L.FP4_MX, 1, 4096) >= 2048 + 32 * 512 + 4


def test_c_entry_points_refuse_before_any_launch():
    import duqlinear4bitcuda_b200.lib as L
    c, MX, NV = L.cdll, L.FP4_MX, L.FP4_NV
    q = c.duq4_fp4_quantize
    assert q(5, 0, P, 4, 64, 64, P, P, P, None) == -3 and q(MX, 2, P, 4, 64, 64, P, P, P, None) == -3
    for cols in (0, 16, 48, 65568):
        assert q(MX, 0, P, 4, cols, 65568, P, P, P, None) == -2
    assert q(MX, 0, P, 4, 64, 32, P, P, P, None) == -2 and q(MX, 0, P, 4, 64, 68, P, P, P, None) == -2
    assert q(NV, 0, P, 4, 64, 64, P, P, None, None) == -1 and q(MX, 0, None, 4, 64, 64, P, P, None, None) == -1
    assert q(MX, 0, P + 2, 4, 64, 64, P, P, None, None) == -5 and q(MX, 0, P, 4, 64, 64, P, P + 8, None, None) == -5
    assert q(MX, 0, None, 0, 64, 64, None, None, None, None) == 0
    s = c.duq4_fp4_silu_mul_quantize
    assert s(NV, 1, P, 4, 64, 128, 60, P, P, P, None) == -2 and s(NV, 1, P, 4, 64, 128, 72, P, P, P, None) == -2
    assert s(NV, 1, P, 4, 64, 100, 32, P, P, P, None) == -2 and s(NV, 1, P, 4, 64, 128, 64, P, None, P, None) == -1
    d = c.duq4_fp4_dequantize
    assert d(MX, 3, P, P, None, 4, 64, P, None) == -3 and d(MX, 0, P, P, None, 4, 40, P, None) == -2
    assert d(NV, 0, P, P, None, 4, 64, P, None) == -1 and d(MX, 0, P + 4, P, None, 4, 64, P, None) == -5
    g = lambda **kw: c.duq4_linear_fp4(*{**dict(f=NV, a=P, sa=P, ra=None, w=P, sw=P, rw=None, m=4, n=8, k=64, b=None, dt=0, o=P, ldo=0, st=None), **kw}.values())
    assert g(f=1) == -3 and g(dt=2) == -3 and g(k=40) == -2 and g(ldo=7) == -2 and g(a=None) == -1 and g(sw=None) == -1 and g(o=None) == -1
    assert g(a=P + 8) == -5 and g(sa=P + 4) == -5 and g(rw=P + 2) == -5 and g(b=P + 1) == -5 and g(m=0) == 0 and g(n=0) == 0
    x = c.duq4_linear_fp4_from_16bit
    assert x(NV, 0, P, P, P, None, 4, 8, 64, None, P, 0, None, 1 << 20, None) == -4
    assert x(NV, 0, P, P, P, None, 4, 8, 64, None, P, 0, P, 100, None) == -4
    assert x(NV, 0, P, P, P, None, 4, 8, 64, None, P, 0, P + 16, 1 << 20, None) == -4


def test_norm_entry_point_refuses_before_any_launch():
    import duqlinear4bitcuda_b200.lib as L
    c = L.cdll

    def call(format=L.FP4_NV, rows=4, cols=64, out=P, scales=P, row_scales=P, **kw):
        n = L.NormResidual()
        for k, v in {**dict(dtype=0, residual_scale=1.0, clip_ratio=1.0, eps=1e-6, x=P, residual=P, residual_out=P, weight=P), **kw}.items():
            setattr(n, k, v)
        return c.duq4_norm_residual_quantize(format, ctypes.byref(n), rows, cols, out, scales, row_scales, None)
    assert c.duq4_norm_residual_quantize(L.FP4_NV, None, 4, 64, P, P, P, None) == -1
    assert call(format=2) == -3 and call(format=L.MODE_SYM, dtype=1) == -3 and call(dtype=2) == -3
    assert call(cols=48) == -2 and call(cols=65568) == -2 and call(eps=-1.0) == -2 and call(eps=float("nan")) == -2
    assert call(x=None) == -1 and call(weight=None) == -1 and call(out=None) == -1 and call(scales=None) == -1 and call(row_scales=None) == -1
    assert call(residual_out=None) == -1 and call(residual=None) == -1
    assert call(residual=None, residual_out=None, gate=P) == -1 and call(residual=None, residual_out=None, post_weight=P) == -1
    assert call(format=L.MODE_ASYM, row_scales=None) == -1
    assert call(gate=P + 2) == -5 and call(residual_out=P + 8) == -5 and call(scales=P + 8) == -5 and call(row_scales=P + 2) == -5
    assert call(rows=0, x=None) == 0


def test_operators_refuse_wrong_arguments():
    import duqlinear4bitcuda_b200._CUDA as o
    x, u, f = torch.zeros(4, 64, dtype=H), torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4)
    s = torch.zeros(512, dtype=torch.uint8)
    for call, match in [
        (lambda: o.fp4_quantize("int4", x), "unknown format"),
        (lambda: o.fp4_quantize("mxfp4", x.float()), "x to have dtype Half or BFloat16"),
        (lambda: o.fp4_quantize("mxfp4", x), "CUDA tensor"),
        (lambda: o.fp4_quantize("mxfp4", x[0]), "2-D"),
        (lambda: o.fp4_silu_mul_quantize("nvfp4", x[:, :63]), "2\\*I"),
        (lambda: o.fp4_dequantize("mxfp4", u.int(), s, None, H), "codes to have dtype"),
        (lambda: o.fp4_dequantize("nvfp4", u, s, f.double(), H), "row_scales to have dtype"),
        (lambda: o.fp4_dequantize("nvfp4", u, s, f, torch.int32), "the result to have dtype"),
        (lambda: o.norm_residual_quantize("nvfp4", x, torch.ones(64, dtype=B)), "weight to have dtype"),
        (lambda: o.norm_residual_quantize("sym", x.to(B), torch.ones(64, dtype=B)), "sym and asym take Half"),
        (lambda: o.norm_residual_quantize("fp8", x, torch.ones(64, dtype=H)), "unknown format"),
        (lambda: o.linear_fp4("mxfp4", u, s, None, u, s, f.half()), "W_row_scales to have dtype"),
        (lambda: o.linear_fp4("mxfp4", u, s, None, u, s, None, torch.ones(4, dtype=B), H), "bias to have dtype"),
        (lambda: o.linear_fp4("mxfp4", u, s, None, u, s, None, None, torch.float32), "the result to have dtype"),
        (lambda: o.linear_fp4_from_16bit("mxfp4", x, u.to(torch.int8), s, None), "W to have dtype"),
        (lambda: o.linear_fp4_from_16bit("mxfp4", x, u, s, None, torch.ones(4)), "bias to have dtype"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()


@pytest.mark.parametrize("rows,blocks", [(1, 1), (3, 4), (127, 5), (130, 9), (256, 8)])
def test_tile_order_of_block_scales(rows, blocks):
    from duqlinear4bitcuda_b200.tools import quantization as qz
    b = np.random.default_rng(rows).integers(0, 256, (rows, blocks), dtype=np.uint8)
    t = qz.fp4_tile_scales(torch.from_numpy(b))
    assert np.array_equal(t.numpy(), F.tile(b))
    assert np.array_equal(qz.fp4_untile_scales(t, rows, blocks).numpy(), b)
    assert np.array_equal(F.untile(t.numpy(), rows, blocks), b)


def test_oracle_against_differences():
    """The oracle's roundings by brute force: no e2m1 (e4m3) number is nearer than the one it takes."""
    a = np.abs(np.random.default_rng(0).standard_normal(4000)) * 3
    assert np.array_equal(np.abs(F.E2M1[F.nearest(a, F.E2M1)] - np.minimum(a, 6)), np.abs(F.E2M1[None] - np.minimum(a, 6)[:, None]).min(1))
    assert list(F.E2M1[F.nearest(np.array([.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 9]), F.E2M1)]) == [0, 1, 1, 2, 2, 4, 4, 6]
    b = a * 60
    assert np.allclose(np.abs(F.E4M3[F.nearest(b, F.E4M3)] - b), np.abs(F.E4M3[None] - b[:, None]).min(1), rtol=0, atol=0)
    assert np.array_equal(F.E4M3[1:], torch.arange(1, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())
    v = np.abs(np.random.default_rng(1).standard_normal(1000)) * 1e-3
    assert np.array_equal(F.bf16(v), torch.from_numpy(v).float().bfloat16().double().numpy())


def test_linear_module_state():
    import qlinear4bit.nn as nn
    m = nn.LinearFP4(96, 40, bias=True, format="nvfp4", dtype=B)
    assert sorted(m.state_dict()) == ["bias", "weight", "weight_row_scales", "weight_scales"]
    assert m.weight.shape == (40, 48) and m.weight_scales.shape == (2 * 512,) and m.bias.dtype == B
    assert sorted(nn.LinearFP4(96, 40, format="mxfp4").state_dict()) == ["weight", "weight_scales"]
    with pytest.raises(ValueError):
        nn.LinearFP4(100, 40)
    with pytest.raises(ValueError):
        nn.QuantizerFP4("sym")
    assert sorted(nn.NormResidualQuantizer(64, "sym", post_norm=True).state_dict()) == ["post_weight", "weight"]
