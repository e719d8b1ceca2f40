"""Launches that begin while the one in front still writes what they read: the integer operators of few tokens behind the fp4
operators that let them in early. Every value as with a wait between the two."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    import duqlinear4bitcuda_b200._CUDA as o
    return o


@pytest.mark.parametrize("rows,cols", [(16, 32), (16, 96), (13, 4096), (16, 16384)])
@pytest.mark.parametrize("kind", ["sym", "asym"])
def test_integer_quantizer_behind_the_reading_back(kind, rows, cols):
    """fp4_dequantize lets the quantizer in at its start and writes x for as long as it runs."""
    o = ops()
    quantize = o.quantize_sym_fused if kind == "sym" else o.quantize_asym_fused
    g = torch.Generator().manual_seed(rows + cols)
    packed = [o.fp4_quantize("nvfp4", torch.randn(rows, cols, generator=g).half().cuda()) for _ in range(4)]
    want = []
    for p in packed:
        x = o.fp4_dequantize("nvfp4", *p, torch.float16)
        torch.cuda.synchronize()
        want.append([t.clone() for t in quantize(x)])
        torch.cuda.synchronize()
    for _ in range(20):
        got = [quantize(o.fp4_dequantize("nvfp4", *p, torch.float16)) for p in packed]
        for a, b in zip(got, want):
            assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("rows,cols", [(16, 32), (15, 96), (16, 4096)])
def test_integer_quantizer_behind_a_stream_updated_in_place(rows, cols):
    """The joint writes the residual stream in place while the quantizer that reads it is resident; neighbouring rows share cache
    lines."""
    import duqlinear4bitcuda_b200.lib as L
    g = torch.Generator().manual_seed(cols)
    x, start = torch.randn(rows, cols, generator=g).half().cuda(), torch.randn(rows, cols, generator=g).half().cuda()
    w, out = torch.ones(cols, dtype=torch.float16, device="cuda"), torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    stream = start.clone()
    n = L.NormResidual()
    n.dtype, n.residual_scale, n.clip_ratio, n.eps = L.DTYPE_F16, 0.5, 1.0, 1e-6
    n.x, n.residual, n.residual_out, n.weight = x.data_ptr(), stream.data_ptr(), stream.data_ptr(), w.data_ptr()

    def steps(wait):
        stream.copy_(start)
        got = []
        for _ in range(30):
            L.call("duq4_norm_residual_quantize", 0, ctypes.byref(n), rows, cols, L.ptr(out), None, None, L.current_stream())
            if wait:
                torch.cuda.synchronize()
            got += ops().quantize_sym_fused(stream)
            if wait:
                torch.cuda.synchronize()
        return got
    want = steps(True)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(steps(False), want))


@pytest.mark.parametrize("static", [0, 1])
@pytest.mark.parametrize("tokens,k,n", [(1, 4096, 4096), (4, 11008, 4096), (16, 4096, 22016), (8, 128, 40), (16, 1024, 300)])
def test_integer_layer_behind_fp4_operators(static, tokens, k, n):
    """joint (codes of the integer format) -> integer product, and reading back -> quantizer -> product, with and without the
    promise on weights: the products' kernels for few tokens read codes that the launch in front has just written."""
    import duqlinear4bitcuda_b200.lib as L
    import duqlinear4bitcuda_b200.nn as nn
    g = torch.Generator().manual_seed(n)
    layer = nn.Linear4bitSQ(k, n).cuda()
    layer.weight.copy_(torch.randint(0, 256, layer.weight.shape, generator=g, dtype=torch.uint8))
    layer.weight_scales.fill_(0.01)
    joint, quantizer = nn.NormResidualQuantizer(k, "sym").cuda(), nn.SymQuantizer()
    xs = [torch.randn(tokens, k, generator=g).half().cuda() for _ in range(4)]
    packed = [nn.QuantizerFP4("mxfp4")(x) for x in xs]

    def run(wait):
        got = []
        for x, p in zip(xs, packed):
            for f in (lambda: joint(x), lambda: quantizer(p.dequantize())):
                q = f()
                if wait:
                    torch.cuda.synchronize()
                got.append(layer(q))
                if wait:
                    torch.cuda.synchronize()
        return got
    old = L.cdll.duq4_set_static_weights(static)
    try:
        want = run(True)
        for _ in range(10):
            assert all(torch.equal(a, b) for a, b in zip(run(False), want))
    finally:
        L.cdll.duq4_set_static_weights(old)
