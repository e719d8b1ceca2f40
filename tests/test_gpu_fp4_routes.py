"""The fp4 product on each of its routes, at sizes that tests/test_fp4_routes_cpu.py holds to them: every element against the
definition in 64 bits, and the layer from 16-bit activations eagerly, captured, and with launches behind it that read its
result."""
import numpy as np
import pytest
import torch

from tests import _fp4 as F
from tests import _fp4_routes as R

pytestmark = pytest.mark.gpu
FORMATS = ["mxfp4", "nvfp4"]
H, B = torch.float16, torch.bfloat16


def ops():
    import duqlinear4bitcuda_b200._CUDA as o
    return o


@pytest.fixture(autouse=True)
def on_the_gpu_the_routes_are_for():
    if torch.cuda.get_device_properties(0).multi_processor_count != R.SMS:
        pytest.skip("the sizes are chosen for 148 SMs")


def operand(fmt, rows, cols, seed, scale=1.0):
    """Random codes and scales on the GPU: ((codes, tiled block scales, row factors), exact doubles)."""
    from duqlinear4bitcuda_b200.tools import quantization as qz
    g = torch.Generator(device="cuda").manual_seed(seed)
    code = torch.randint(0, 256, (rows, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
    lo, hi = (120, 130) if fmt == "mxfp4" else (8, 0x7F)
    byte = torch.randint(lo, hi, (rows, cols // F.BLOCK[fmt]), generator=g, device="cuda", dtype=torch.uint8)
    row = (0.25 + torch.rand(rows, generator=g, device="cuda")) * (scale if fmt == "mxfp4" else scale * 0.01)
    grid = torch.from_numpy(np.concatenate([F.E2M1, -F.E2M1])).cuda()
    v = grid[torch.stack([code & 15, code >> 4], -1).view(rows, cols).int()]
    s = torch.exp2(byte.double() - 127) if fmt == "mxfp4" else torch.from_numpy(F.E4M3).cuda()[byte.int()]
    return (code, qz.fp4_tile_scales(byte), row), v * (s * row.double()[:, None]).repeat_interleave(F.BLOCK[fmt], 1)


def check(got, a, w, bias):
    """Half a step of the type and, for the 32-bit sum, at most one rounding or cut of 2^-23 per addition of the sum of
    magnitudes, a few more for the factors."""
    exact, mags = a @ w.T, a.abs() @ w.abs().T
    if bias is not None:
        exact, mags = exact + bias.double(), mags + bias.double().abs()
    tol = torch.finfo(got.dtype).eps / 2 * exact.abs() * (1 + 2.0 ** -7) + (a.shape[1] + 8) * 2.0 ** -23 * mags
    if got.dtype == H:
        tol += 2.0 ** -25
    off = (got.double() - exact).abs()
    assert bool((off <= tol).all()), ((off / tol).max().item(), (off > tol).nonzero()[:5].tolist())


ALL = R.PAIR_ROUNDS + R.TWO_LAUNCHES + R.FEW_TOKEN_BLOCKS + R.PAIR_ONE_ROUND


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", ALL)
def test_every_element(fmt, m, n, k):
    dtype = B if (m + n) % 2 else H
    a, av = operand(fmt, m, k, m, 1.0 if dtype == B else 2.0 ** -12)
    w, wv = operand(fmt, n, k, n)
    bias = torch.randn(n, device="cuda").to(dtype) if k % 64 == 32 else None
    args = (fmt, *a, *w, bias, dtype)
    got = ops().linear_fp4(*args)
    check(got, av, wv, bias)
    assert torch.equal(ops().linear_fp4(*args), got)


def layer(fmt, m, n, k, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w, _ = operand(fmt, n, k, seed + 1, 2.0 ** -8)
    return x, w, torch.randn(n, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", ALL)
def test_from_16bit_equals_quantizer_and_product(fmt, m, n, k):
    dtype = H if (m + n) % 2 else B
    x, w, bias = layer(fmt, m, n, k, dtype)
    q = ops().fp4_quantize(fmt, x)
    torch.cuda.synchronize()
    want = ops().linear_fp4(fmt, *q, *w, bias, dtype)
    torch.cuda.synchronize()
    for _ in range(5):
        assert torch.equal(ops().linear_fp4_from_16bit(fmt, x, *w, bias), want)


@pytest.mark.parametrize("static", [0, 1])
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [R.TWO_LAUNCHES[0], (1100, 13024, 3104), (300, 9600, 1056)])
def test_launches_behind_read_the_whole_result(fmt, m, n, k, static):
    """quantizer -> product (its second launch too) -> quantizer, joint in place of nothing, product on top, eagerly and captured
    twice and replayed in turn: as with a wait after every call."""
    import duqlinear4bitcuda_b200.lib as L
    x, w, bias = layer(fmt, m, n, k, B)
    w2, _ = operand(fmt, 200, n, 5, 2.0 ** -8)
    norm = torch.ones(n, device="cuda", dtype=B)

    def run(x, wait=False):
        pause = torch.cuda.synchronize if wait else lambda: None
        y = ops().linear_fp4_from_16bit(fmt, x, *w, bias)
        pause()
        q = ops().fp4_quantize(fmt, y)
        pause()
        z = ops().linear_fp4(fmt, *q, *w2, None, B)
        pause()
        r, *h = ops().norm_residual_quantize(fmt, y, norm, 1e-6, y, None, None, 0.5)
        pause()
        y2 = ops().linear_fp4_from_16bit(fmt, x.flip(0).contiguous(), *w, bias)
        pause()
        return y, q[0], z, r, h[0], y2
    assert 0 < L.cdll.duq4_linear_fp4_pair_columns(m, n, k, R.SMS) < n or (m, n, k) != R.TWO_LAUNCHES[0]
    old = L.cdll.duq4_set_static_weights(static)
    try:
        xs = [x, x.roll(1, 0).contiguous()]
        want = [[t.clone() for t in run(x, True)] for x in xs]
        for _ in range(3):
            for x, ws in zip(xs, want):
                assert all(torch.equal(a, b) for a, b in zip(run(x), ws))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(xs[0])
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for x in xs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = run(x)
            graphs.append((g, out))
        for _ in range(3):
            for g, out in graphs:
                out[0].zero_()
                g.replay()
        torch.cuda.synchronize()
        for (_, out), ws in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, ws))
    finally:
        L.cdll.duq4_set_static_weights(old)


@pytest.mark.parametrize("fmt", FORMATS)
def test_routes_side_by_side(fmt):
    """The routes on streams of their own at once: pair rounds, two launches, few tokens, one token."""
    jobs = []
    for i, (m, n, k) in enumerate([R.PAIR_ROUNDS[2], R.TWO_LAUNCHES[0], R.FEW_TOKEN_BLOCKS[0], (1, 4096, 4096)]):
        x, w, bias = layer(fmt, m, n, k, B, i)
        jobs.append(((fmt, x, *w, bias), ops().linear_fp4_from_16bit(fmt, x, *w, bias), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for args, want, s in jobs:
            with torch.cuda.stream(s):
                outs.append((ops().linear_fp4_from_16bit(*args), want))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)


def test_beside_the_integer_products():
    """fp4 and integer products on streams of their own: kernels that take all of TMEM, some of it and clusters that wait for one
    another meet on the same SMs."""
    import ctypes
    import duqlinear4bitcuda_b200.lib as L
    jobs = []
    for i, (m, n, k) in enumerate([(64, 22016, 1024), (100, 4096, 4096), (512, 8192, 2048), (48, 9472, 512)]):
        g = torch.Generator(device="cuda").manual_seed(i)
        a, w = (torch.randint(0, 256, (r, k // 2), generator=g, device="cuda", dtype=torch.uint8) for r in (m, n))
        sa, sw = (torch.rand(r, generator=g, device="cuda").half() * 0.01 for r in (m, n))
        jobs.append((lambda a=a, w=w, sa=sa, sw=sw: ops().linear_w4a4("sym", a, w, sa, None, sw)))
    for i, (fmt, m, n, k) in enumerate([("nvfp4", 4, 2048, 1024), ("mxfp4", 16, 1024, 2048), ("nvfp4", 40, 4096, 512), ("mxfp4", 128, 4096, 4096),
                                        ("nvfp4", 300, 3000, 1056), ("mxfp4", 1, 9000, 96)]):
        x, w, bias = layer(fmt, m, n, k, B, i)
        jobs.append((lambda fmt=fmt, x=x, w=w, bias=bias: ops().linear_fp4_from_16bit(fmt, x, *w, bias)))
    want = [j() for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    outs = []
    for r in range(30):
        for i in range(len(jobs)):
            i = (i * 3 + r) % len(jobs)
            with torch.cuda.stream(streams[i]):
                outs.append((jobs[i](), want[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)
    status = ctypes.c_int32(-1)
    L.call("duq4_last_device_status", L.current_stream(), ctypes.byref(status))
    assert status.value == 0
