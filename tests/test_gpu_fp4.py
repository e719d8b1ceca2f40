"""Microscaled 4-bit operators against their definitions in 64 bits (tests/_fp4.py)."""
import numpy as np
import pytest
import torch

from tests import _fp4 as F

pytestmark = pytest.mark.gpu
FORMATS = ["mxfp4", "nvfp4"]
DTYPES = [torch.float16, torch.bfloat16]


def ops():
    import duqlinear4bitcuda_b200._CUDA as o
    return o


def make(rows, cols, dtype, seed=0, loud=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g)
    if loud:
        x = x * torch.where(torch.rand(cols, generator=g) < 0.02, 30.0, 1.0) * torch.exp(torch.randn(rows, 1, generator=g))
    return x.to(dtype)


def check_quantized(fmt, got, x64):
    """Codes, block scales (in place and zero in the padding columns) and row scales are those of the definition, exactly."""
    codes, tiled, rows = got
    c, b, r = F.quantize(fmt, x64)
    n, blocks = b.shape
    g = codes.cpu().numpy()
    t = tiled.cpu().numpy()
    assert np.array_equal(F.untile(t, n, blocks), b)
    padded = -(-blocks // 4) * 4
    assert not F.untile(t, n, padded)[:, blocks:].any()
    assert np.array_equal(F.unpack(g), c)
    if fmt == "nvfp4":
        assert np.array_equal(rows.cpu().numpy().astype(np.float64), r)
    else:
        assert rows is None


SIZES = [(1, 32), (1, 4096), (3, 64), (5, 96), (128, 160), (129, 224), (33, 2080), (7, 8192), (2, 11008), (3, 16416), (2, 33024), (1, 65536)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_quantize(fmt, dtype, rows, cols):
    x = make(rows, cols, dtype, rows + cols)
    check_quantized(fmt, ops().fp4_quantize(fmt, x.cuda()), x.double().numpy())


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_every_half(fmt):
    """Every finite fp16 number as an element, beside tops of every exponent: all roundings and ties."""
    bits = torch.arange(0, 0x7C00, dtype=torch.int32)
    x = bits.to(torch.int16).view(torch.float16)
    x = torch.cat([x, -x])[:63488].reshape(-1, 64).clone()
    x = torch.cat([x, x[torch.randperm(x.shape[0], generator=torch.Generator().manual_seed(1))].reshape(64, -1).t().contiguous().view(-1, 64)])
    check_quantized(fmt, ops().fp4_quantize(fmt, x.cuda()), x.double().numpy())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_special_rows(fmt, dtype):
    """Zero rows and blocks, the smallest and largest numbers, infinities and NaNs: a bad block reads back as NaN, the others
    of its row as if it were zero."""
    x = make(12, 256, dtype, 3)
    x[0] = 0
    x[1] = 0
    x[1, 255] = torch.finfo(dtype).smallest_normal
    x[2] = torch.finfo(dtype).max
    x[3, :16] = 0
    x[4, 5] = float("inf")
    x[5, 40] = float("nan")
    x[6, 70] = -float("inf")
    x[7] = float("nan")
    x[8] = -torch.finfo(dtype).tiny * torch.finfo(dtype).eps   # the smallest subnormal
    x[9] = torch.finfo(dtype).smallest_normal
    x[10, ::2] = -0.0
    got = ops().fp4_quantize(fmt, x.cuda())
    check_quantized(fmt, got, x.double().numpy())
    back = ops().fp4_dequantize(fmt, *got, torch.float32).cpu()
    want = torch.from_numpy(F.values(fmt, *F.quantize(fmt, x.double().numpy())).astype(np.float32))
    assert torch.equal(back.isnan(), want.isnan())
    assert torch.allclose(back.nan_to_num(), want.nan_to_num(), rtol=2 ** -22, atol=0)
    assert back[4, :16].isnan().all() and not back[4, 32:].isnan().any()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (130, 96), (5, 4128)])
def test_dequantize(fmt, dtype, rows, cols):
    packed, tiled, row, v = F.random_operand(fmt, rows, cols, rows)
    if fmt == "mxfp4":
        row, v = None, v / row[:, None]
    got = ops().fp4_dequantize(fmt, F.cuda(packed), F.cuda(tiled), F.cuda(row), dtype).double().cpu().numpy()
    # half a step of the result's type on top of the one rounding of block scale * row scale and of its product
    tol = torch.finfo(dtype).eps / 2 + 2 * 2.0 ** -24
    assert np.all(np.abs(got - v) <= tol * np.abs(v) * (1 + 2.0 ** -10) + (2.0 ** -25 if dtype == torch.float16 else 0))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,inter", [(1, 32), (16, 11008), (131, 96), (3, 28672)])
def test_silu_mul_quantize_equals_the_composition(fmt, dtype, rows, inter):
    gu = (make(rows, 2 * inter, dtype, 5, loud=False) * 2).cuda()
    h = torch.nn.functional.silu(gu[:, :inter]) * gu[:, inter:]
    a, b = ops().fp4_silu_mul_quantize(fmt, gu), ops().fp4_quantize(fmt, h)
    assert torch.equal(a[0], b[0])
    blocks = inter // F.BLOCK[fmt]
    assert np.array_equal(F.untile(a[1].cpu().numpy(), rows, blocks), F.untile(b[1].cpu().numpy(), rows, blocks))
    assert a[2] is None if fmt == "mxfp4" else torch.equal(a[2], b[2])


def _norm(t, w, eps):
    """fp32 steps of x * rms(x) * w with the mean in 64 bits."""
    d = t.double()
    rstd = (1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)).float()
    return t.float() * rstd * w.float()


def _joint(x, weight, eps, residual, post, gate, scale):
    y = x.float()
    if residual is None:
        r = x
    else:
        if post is not None:
            y = _norm(x, post, eps)
        if gate is not None:
            y = y * gate.float()
        r = (residual.float() + y * scale).to(x.dtype)
    return r, _norm(r, weight, eps).to(x.dtype)


@pytest.mark.parametrize("fmt", ["none", "sym", "asym", "mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (5, 96), (130, 2080), (3, 8192), (2, 16448), (1, 65536)])
@pytest.mark.parametrize("form", ["pre", "residual", "post", "gate", "gate_row", "all"])
def test_norm_residual_quantize_equals_its_steps(fmt, dtype, rows, cols, form):
    if fmt in ("sym", "asym") and (dtype != torch.float16 or cols > 32768):
        pytest.skip("integer formats: fp16, and the quantizer compared with takes 32768 columns in the same arithmetic")
    x, residual = make(rows, cols, dtype, 1).cuda(), make(rows, cols, dtype, 2).cuda()
    weight, post = (1 + 0.1 * make(1, cols, torch.float32, 3, False)[0]).to(dtype).cuda(), make(1, cols, dtype, 4, False)[0].cuda()
    gate = make(rows, cols, dtype, 5, False).cuda() if form == "gate_row" else make(1, cols, dtype, 6, False)[0].cuda()
    res = None if form == "pre" else residual
    post = post if form in ("post", "all") else None
    gate = gate if form in ("gate", "gate_row", "all") else None
    scale = 1.0 if form in ("pre", "residual") else 0.37
    r, h = _joint(x, weight, 1e-5, res, post, gate, scale)
    got_r, *got = ops().norm_residual_quantize(fmt, x, weight, 1e-5, res, post, gate, scale)
    assert got_r is None if res is None else torch.equal(got_r, r)
    if fmt == "none":
        assert torch.equal(got[0], h)
        return
    want = {"sym": lambda: ops().quantize_sym_fused(h), "asym": lambda: ops().quantize_asym_fused(h)}.get(fmt, lambda: ops().fp4_quantize(fmt, h))()
    assert torch.equal(got[0], want[0])
    if fmt in ("sym", "asym"):
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))
        return
    blocks = cols // F.BLOCK[fmt]
    assert np.array_equal(F.untile(got[1].cpu().numpy(), rows, blocks), F.untile(want[1].cpu().numpy(), rows, blocks))
    assert got[2] is None if fmt == "mxfp4" else torch.equal(got[2], want[2])


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_of_extreme_rows(dtype):
    """Rows of zeros, of the smallest and the largest numbers, with an infinity, with a NaN."""
    big = torch.finfo(dtype).max
    x = torch.zeros(6, 96, dtype=dtype)
    x[1] = torch.finfo(dtype).smallest_normal
    x[2] = big
    x[3] = make(1, 96, dtype)[0]
    x[3, 7] = float("inf")
    x[4] = make(1, 96, dtype)[0]
    x[4, 90] = float("nan")
    x[5] = torch.linspace(-1, 1, 96).to(dtype) * (big / 4)
    w = torch.ones(96, dtype=dtype)
    for eps in (0.0, 1e-6):
        want = _joint(x, w, eps, None, None, None, 1.0)[1]
        got = ops().norm_residual_quantize("none", x.cuda(), w.cuda(), eps)[1].cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(), want.nan_to_num())


def check_product(got, a, w, bias, dtype):
    """|y - exact| within half a step of the type and the rounding of a 32-bit sum of K products: each product of two codes and
    the sum's terms are exact, the terms' running sum is rounded (or cut off) at most once per addition, so the error is
    at most K steps of 2^-23 of the sum of magnitudes; a few more roundings for the factors."""
    exact = a @ w.T + (0 if bias is None else bias)
    mags = np.abs(a) @ np.abs(w).T + (0 if bias is None else np.abs(bias))
    k = a.shape[1]
    tol = torch.finfo(dtype).eps / 2 * np.abs(exact) * (1 + 2.0 ** -7) + (k + 8) * 2.0 ** -23 * mags
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    off = np.abs(got.double().cpu().numpy() - exact)
    assert np.all(off <= tol), (np.nanmax(off / tol), np.argwhere(~(off <= tol))[:5])


PRODUCTS = [(1, 8, 32), (1, 129, 96), (2, 256, 256), (3, 100, 288), (8, 1024, 512), (16, 130, 4096), (17, 33, 1056), (32, 512, 11008), (33, 384, 640),
            (77, 300, 1120), (128, 256, 1024), (129, 257, 544), (200, 1000, 320), (256, 512, 2048), (300, 384, 64), (513, 700, 96), (640, 640, 1312)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("form", ["plain", "rows", "bias"])
def test_linear_fp4(fmt, m, n, k, form):
    dtype = torch.bfloat16 if (m + n) % 2 else torch.float16
    ap, at, ar, av = F.random_operand(fmt, m, k, m + n + k, form != "plain")
    wp, wt, wr, wv = F.random_operand(fmt, n, k, m * n + k, form != "plain")
    scale = 1.0 if dtype == torch.bfloat16 else 2.0 ** -12   # results inside fp16
    if form == "plain" and dtype == torch.float16:
        wr, wv = np.full(n, scale / (1 if fmt == "mxfp4" else 64), np.float32), wv * (scale / (1 if fmt == "mxfp4" else 64))
    elif dtype == torch.float16 and fmt == "mxfp4":
        wr, wv = wr * np.float32(scale), wv * scale
    bias = make(1, n, dtype, 9)[0] if form == "bias" else None
    got = ops().linear_fp4(fmt, F.cuda(ap), F.cuda(at), F.cuda(ar), F.cuda(wp), F.cuda(wt), F.cuda(wr), None if bias is None else bias.cuda(), dtype)
    assert got.shape == (m, n) and got.dtype == dtype
    check_product(got, av, wv, None if bias is None else bias.double().numpy(), dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (5, 70, 96), (16, 640, 1024), (40, 512, 512), (150, 384, 1376), (520, 1030, 512)])
def test_linear_from_16bit_equals_quantizer_and_product(fmt, dtype, m, n, k):
    x = make(m, k, dtype, 7).cuda()
    wp, wt, wr, _ = F.random_operand(fmt, n, k, 11)
    w = (F.cuda(wp), F.cuda(wt), F.cuda(wr))
    bias = make(1, n, dtype, 9)[0].cuda()
    want = ops().linear_fp4(fmt, *ops().fp4_quantize(fmt, x), *w, bias, dtype)
    assert torch.equal(ops().linear_fp4_from_16bit(fmt, x, *w, bias), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [3, 150])
def test_a_bad_token_spoils_its_own_row_only(fmt, m):
    """Infinities and NaNs in one token's activations: its row of the result is NaN, every other row as without them."""
    x = make(m, 256, torch.bfloat16, 7).cuda()
    wp, wt, wr, _ = F.random_operand(fmt, 200, 256, 11)
    w = (F.cuda(wp), F.cuda(wt), F.cuda(wr))
    clean = ops().linear_fp4_from_16bit(fmt, x, *w)
    x[1, 100], x[2, 3] = float("nan"), float("-inf")
    got = ops().linear_fp4_from_16bit(fmt, x, *w)
    assert got[1:3].isnan().all()
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])


def test_empty_batches():
    o = ops()
    for fmt in FORMATS:
        x = torch.empty(0, 64, dtype=torch.float16, device="cuda")
        q = o.fp4_quantize(fmt, x)
        assert q[0].shape == (0, 32) and o.fp4_dequantize(fmt, *q, torch.float16).shape == (0, 64)
        wp, wt, wr, _ = F.random_operand(fmt, 40, 64, 1)
        assert o.linear_fp4_from_16bit(fmt, x, F.cuda(wp), F.cuda(wt), F.cuda(wr)).shape == (0, 40)
        assert o.norm_residual_quantize(fmt, x, torch.ones(64, dtype=torch.float16, device="cuda"))[1].shape == (0, 32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("lead", [(0,), (2, 0), (0, 3)])
def test_modules_on_empty_batches(fmt, lead):
    import duqlinear4bitcuda_b200.nn as nn
    x = torch.empty(*lead, 64, dtype=torch.float16, device="cuda")
    layer = nn.LinearFP4.from_linear(torch.nn.Linear(64, 40, bias=True).half().cuda(), fmt)
    q = nn.QuantizerFP4(fmt)(x)
    assert q.size() == (*lead, 32) and q.dequantize().shape == x.shape
    assert layer(x).shape == (*lead, 40) and layer(q).shape == (*lead, 40)
    assert nn.SiluMulQuantizerFP4(fmt)(x).size() == (*lead, 16)
    for form in (fmt, "sym", "asym", "none"):
        out, stream = nn.NormResidualQuantizer(64, form, post_norm=True).cuda()(x, x, x)
        assert stream.shape == x.shape
        if form == "none":
            assert out.shape == x.shape
        else:
            assert out.size() == (*lead, 32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 19, 300])
def test_mlp_block_of_modules(fmt, tokens):
    """The operators as they are used: norm -> gate/up layer -> SiLU product -> down layer -> norm after the block, residual
    sum, next norm, quantized. Every stage equals the same stage from its 16-bit or read-back inputs; graph replay too."""
    import duqlinear4bitcuda_b200.nn as nn
    g = torch.Generator().manual_seed(tokens)
    dim, inter, dtype = 256, 416, torch.bfloat16
    lin = lambda i, o: torch.nn.Linear(i, o, bias=True).to(dtype).cuda()
    gate_up, down = lin(dim, 2 * inter), lin(inter, dim)
    first, last = nn.NormResidualQuantizer(dim, fmt, dtype=dtype).cuda(), nn.NormResidualQuantizer(dim, fmt, post_norm=True, residual_scale=0.5, dtype=dtype).cuda()
    q_gate_up, q_down = nn.LinearFP4.from_linear(gate_up, fmt, dtype), nn.LinearFP4.from_linear(down, fmt, dtype)
    glue = nn.SiluMulQuantizerFP4(fmt)
    x = torch.randn(1, tokens, dim, generator=g).to(dtype).cuda()
    gate = torch.randn(1, tokens, dim, generator=g).to(dtype).cuda()

    def block(x):
        h = first(x)
        y = q_gate_up(h)
        a = glue(y)
        z = q_down(a)
        return h, y, a, z, *last(z, x, gate)
    h, y, a, z, nxt, stream = block(x)
    assert nxt.size() == (1, tokens, dim // 2) and stream.shape == x.shape
    assert torch.equal(q_gate_up(first(x)), y)
    check_product(y[0], h.dequantize(torch.float32)[0].double().cpu().numpy(),
                  _weights64(q_gate_up), q_gate_up.bias.double().cpu().numpy(), dtype)
    check_product(z[0], a.dequantize(torch.float32)[0].double().cpu().numpy(), _weights64(q_down), q_down.bias.double().cpu().numpy(), dtype)
    r, hn = _joint(z[0], last.weight, last.eps, x[0], last.post_weight, gate[0], 0.5)
    assert torch.equal(stream[0], r)
    assert torch.equal(nxt.codes[0], ops().fp4_quantize(fmt, hn)[0])
    # two captures replayed in turn give the eager results
    xs, outs, graphs = [x.clone(), x.flip(-1).contiguous()], [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x)
    torch.cuda.current_stream().wait_stream(side)
    for t in xs:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = block(t)
            outs.append((res[3], res[5], res[4].codes))
        graphs.append(gr)
    for _ in range(2):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for t, got in zip(xs, outs):
        want = block(t)
        assert torch.equal(got[0], want[3]) and torch.equal(got[1], want[5]) and torch.equal(got[2], want[4].codes)


def _weights64(layer):
    rows, cols = layer.out_features, layer.in_features
    byte = F.untile(layer.weight_scales.cpu().numpy(), rows, cols // F.BLOCK[layer.format])
    row = None if layer.weight_row_scales is None else layer.weight_row_scales.cpu().numpy()
    return F.values(layer.format, F.unpack(layer.weight.cpu().numpy()), byte, row)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(300, 9600, 4128), (600, 6500, 2080), (1000, 19001, 288)])
def test_linear_whole_rounds_and_a_rest(fmt, dtype, m, n, k):
    """Problems of more tiles than there are SM pairs, with columns left over behind whole rounds: rows and columns all over
    the result against the definition, and a second call gives the same bits."""
    ap, at, ar, av = F.random_operand(fmt, m, k, 1)
    wp, wt, wr, wv = F.random_operand(fmt, n, k, 2)
    if dtype == torch.float16:
        wr, wv = wr * np.float32(2.0 ** -12), wv * 2.0 ** -12
    args = [fmt, F.cuda(ap), F.cuda(at), F.cuda(ar), F.cuda(wp), F.cuda(wt), F.cuda(wr), None, dtype]
    got = ops().linear_fp4(*args)
    assert torch.equal(ops().linear_fp4(*args), got)
    rows = sorted({0, 1, 127, 128, 255, 256, m // 2, m - 2, m - 1})
    check_product(got[rows], av[rows], wv, None, dtype)
    cols = sorted({0, 255, 256, n // 2, n - 513, n - 257, n - 256, n - 129, n - 1})
    check_product(got[:, cols], av, wv[cols], None, dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("form", ["plain", "bias and strides"])
def test_linear_a_rest_worth_a_second_launch(fmt, form):
    """Long rows and few tiles behind the whole rounds: the columns that are left are another kernel's launch. Columns on both sides
    of the seam, the last ones, and rows that are farther apart than they are long, against the definition."""
    import duqlinear4bitcuda_b200.lib as L
    m, n, k, dtype = 1000, 4994, 8224, torch.bfloat16
    ap, at, ar, av = F.random_operand(fmt, m, k, 1)
    wp, wt, wr, wv = F.random_operand(fmt, n, k, 2)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(3)).to(dtype) if form != "plain" else None
    a, w = [F.cuda(t) for t in (ap, at, ar)], [F.cuda(t) for t in (wp, wt, wr)]
    if bias is None:
        got = ops().linear_fp4(fmt, *a, *w, None, dtype)
    else:
        bias = bias.cuda()
        ld = n + 3
        room = torch.full((m, ld), 77.0, dtype=dtype, device="cuda")
        ptr = lambda t: t.data_ptr()
        assert L.cdll.duq4_linear_fp4(L.FP4_MX if fmt == "mxfp4" else L.FP4_NV, *map(ptr, a), *map(ptr, w), m, n, k, ptr(bias), L.DTYPE_BF16, ptr(room), ld,
                                      torch.cuda.current_stream().cuda_stream) == 0
        assert (room[:, n:] == 77).all()
        got = room[:, :n]
    b64 = None if bias is None else bias.double().cpu().numpy()
    rows = [0, 1, 127, 128, 255, 256, 767, 768, 998, 999]
    check_product(got[rows], av[rows], wv, b64, dtype)
    cols = sorted(set(range(0, n, 256)) | set(range(255, n, 256)) | {n - 1})
    check_product(got[:, cols], av, wv[cols], None if b64 is None else b64[cols], dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(20000, 96), (5000, 1056), (1500, 8192), (700, 16416), (400, 28672), (160, 65536)])
def test_many_rows(fmt, rows, cols):
    """More rows than CTAs fit, so that a CTA does several: the first, the last and some between against the definition, the SiLU
    product and the norm (in place too) against their steps."""
    dtype = torch.bfloat16 if rows % 400 else torch.float16
    x = make(rows, cols, dtype, rows)
    pick = sorted({0, 1, rows // 3, rows // 2, 591, 592, 593, rows - 2, rows - 1} & set(range(rows)))
    codes, tiled, row = ops().fp4_quantize(fmt, x.cuda())
    c, b, r = F.quantize(fmt, x[pick].double().numpy())
    assert np.array_equal(F.unpack(codes.cpu().numpy()[pick]), c)
    assert np.array_equal(F.untile(tiled.cpu().numpy(), rows, cols // F.BLOCK[fmt])[pick], b)
    assert fmt == "mxfp4" or np.array_equal(row.cpu().numpy()[pick].astype(np.float64), r)
    xs = x.cuda()
    gu = torch.cat([xs, xs.flip(0)], 1)
    h = torch.nn.functional.silu(xs) * xs.flip(0)
    same(fmt, ops().fp4_silu_mul_quantize(fmt, gu), ops().fp4_quantize(fmt, h), rows, cols)
    w = (1 + 0.1 * make(1, cols, torch.float32, 3, False)[0]).to(dtype).cuda()
    for post in (None, w.flip(0)):
        r, h = _joint(xs, w, 1e-5, xs.flip(0), post, None, 0.5)
        got = ops().norm_residual_quantize(fmt, xs, w, 1e-5, xs.flip(0), post, None, 0.5)
        assert torch.equal(got[0], r)
        same(fmt, got[1:], ops().fp4_quantize(fmt, h), rows, cols)
    h = _joint(xs, w, 1e-5, None, None, None, 1.0)[1]
    same(fmt, ops().norm_residual_quantize(fmt, xs, w, 1e-5)[1:], ops().fp4_quantize(fmt, h), rows, cols)


def same(fmt, a, b, rows, cols):
    assert torch.equal(a[0], b[0])
    blocks = cols // F.BLOCK[fmt]
    assert np.array_equal(F.untile(a[1].cpu().numpy(), rows, blocks), F.untile(b[1].cpu().numpy(), rows, blocks))
    assert a[2] is None if fmt == "mxfp4" else torch.equal(a[2], b[2])


@pytest.mark.parametrize("rows,cols", [(3, 256), (900, 8192)])
@pytest.mark.parametrize("into", ["residual", "x"])
def test_norm_in_place(rows, cols, into):
    """residual_out may be the residual or x itself (C entry point)."""
    import ctypes
    import duqlinear4bitcuda_b200.lib as L
    x, residual = make(rows, cols, torch.bfloat16, 1).cuda(), make(rows, cols, torch.bfloat16, 2).cuda()
    w = (1 + 0.1 * make(1, cols, torch.float32, 3, False)[0]).to(torch.bfloat16).cuda()
    r, h = _joint(x, w, 1e-6, residual, w, w, 0.25)
    n = L.NormResidual()
    n.dtype, n.residual_scale, n.clip_ratio, n.eps = L.DTYPE_BF16, 0.25, 1.0, 1e-6
    n.x, n.residual, n.post_weight, n.gate, n.weight = x.data_ptr(), residual.data_ptr(), w.data_ptr(), w.data_ptr(), w.data_ptr()
    target = residual if into == "residual" else x
    n.residual_out = target.data_ptr()
    out = torch.empty_like(x)
    L.call("duq4_norm_residual_quantize", 0, ctypes.byref(n), rows, cols, L.ptr(out), None, None, L.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(target, r) and torch.equal(out, h)
    status = ctypes.c_int32(-1)
    L.call("duq4_last_device_status", L.current_stream(), ctypes.byref(status))
    assert status.value == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("rows,cols", [(296, 32), (301, 96), (297, 128), (4001, 160), (1003, 256), (999, 288), (12345, 512)])
def test_narrow_rows(fmt, rows, cols):
    """Several rows a warp, ragged ends: all rows against the definition, the SiLU product and the norm against their steps, and
    nothing written behind the last row."""
    dtype = torch.float16 if rows % 2 else torch.bfloat16
    x = make(rows, cols, dtype, rows)
    x[rows // 2] = 0
    x[rows - 1, 3] = float("inf")
    got = ops().fp4_quantize(fmt, x.cuda())
    check_quantized(fmt, got, x.double().numpy())
    xs = x.cuda()
    xs[rows - 1, 3] = 1
    gu = torch.cat([xs, xs.flip(0)], 1)
    same(fmt, ops().fp4_silu_mul_quantize(fmt, gu), ops().fp4_quantize(fmt, torch.nn.functional.silu(xs) * xs.flip(0)), rows, cols)
    w = (1 + 0.1 * make(1, cols, torch.float32, 3, False)[0]).to(dtype).cuda()
    r, h = _joint(xs, w, 1e-5, xs.flip(0), w.flip(0), xs, 0.5)
    got = ops().norm_residual_quantize(fmt, xs, w, 1e-5, xs.flip(0), w.flip(0), xs, 0.5)
    assert torch.equal(got[0], r)
    same(fmt, got[1:], ops().fp4_quantize(fmt, h), rows, cols)


@pytest.mark.parametrize("fmt,rows,cols", [("mxfp4", 300, 96), ("nvfp4", 333, 160), ("nvfp4", 130, 4128), ("mxfp4", 5, 64)])
def test_quantizer_leaves_what_is_not_its_own(fmt, rows, cols):
    """Rows read with a stride; codes, scales and row scales behind the last row stay as they were, scale bytes of rows that do
    not exist too."""
    import duqlinear4bitcuda_b200.lib as L
    wide = make(rows, cols + 8, torch.bfloat16, 4).cuda()
    f = L.FP4_MX if fmt == "mxfp4" else L.FP4_NV
    size = L.cdll.duq4_fp4_scale_bytes(f, rows, cols)
    codes = torch.full((rows * cols // 2 + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((size + 512,), 0xA5, dtype=torch.uint8, device="cuda")
    row = torch.full((rows + 8,), -7.0, device="cuda")
    L.call("duq4_fp4_quantize", f, L.DTYPE_BF16, L.ptr(wide), rows, cols, cols + 8, L.ptr(codes), L.ptr(scales), L.ptr(row), L.current_stream())
    want = ops().fp4_quantize(fmt, wide[:, :cols].contiguous())
    assert torch.equal(codes[:rows * cols // 2].view(rows, -1), want[0]) and (codes[rows * cols // 2:] == 0xA5).all()
    assert (scales[size:] == 0xA5).all() and (row[rows:] == -7).all()
    padded = -(-(cols // F.BLOCK[fmt]) // 4) * 4
    t = F.untile(scales[:size].cpu().numpy(), -(-rows // 128) * 128, padded)
    assert (t[rows:] == 0xA5).all() and np.array_equal(t[:rows], F.untile(want[1].cpu().numpy(), rows, padded))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 2, 64), (5, 7, 96), (129, 1, 288), (300, 3, 1056), (257, 255, 32), (16, 4096, 65536)])
def test_linear_smallest_and_longest(fmt, m, n, k):
    ap, at, ar, av = F.random_operand(fmt, m, k, 1)
    wp, wt, wr, wv = F.random_operand(fmt, n, k, 2)
    got = ops().linear_fp4(fmt, F.cuda(ap), F.cuda(at), F.cuda(ar), F.cuda(wp), F.cuda(wt), F.cuda(wr), None, torch.bfloat16)
    check_product(got, av, wv, None, torch.bfloat16)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [3, 300])
def test_linear_writes_its_rows_and_columns_only(fmt, m):
    """A result with a row stride inside a larger buffer, rows aligned and not; what lies around it stays."""
    import duqlinear4bitcuda_b200.lib as L
    n, k = 520, 288
    ap, at, ar, _ = F.random_operand(fmt, m, k, 1)
    wp, wt, wr, _ = F.random_operand(fmt, n, k, 2)
    a, w = [F.cuda(t) for t in (ap, at, ar)], [F.cuda(t) for t in (wp, wt, wr)]
    want = ops().linear_fp4(fmt, *a, *w, None, torch.bfloat16)
    f = L.FP4_MX if fmt == "mxfp4" else L.FP4_NV
    for ldo, first in ((536, 16), (544, 8), (523, 1)):
        buf = torch.full((m + 2, ldo), 7.0, dtype=torch.bfloat16, device="cuda")
        L.call("duq4_linear_fp4", f, *map(L.ptr, a), *map(L.ptr, w), m, n, k, None, L.DTYPE_BF16, buf.data_ptr() + 2 * (ldo + first), ldo, L.current_stream())
        flat = buf.view(-1)
        got = torch.as_strided(flat, (m, n), (ldo, 1), ldo + first)
        assert torch.equal(got, want)
        got.fill_(7.0)
        assert (buf == 7).all()


def test_two_streams_and_threads_at_once():
    """Products of both kernels and quantizers queued on several streams by several host threads: every result as alone."""
    import threading
    jobs = []
    for i, (fmt, m, n, k) in enumerate([("nvfp4", 4, 4096, 2048), ("mxfp4", 100, 1000, 4096), ("nvfp4", 700, 2000, 1024), ("mxfp4", 128, 512, 8192)]):
        x = make(m, k, torch.bfloat16, i).cuda()
        wp, wt, wr, _ = F.random_operand(fmt, n, k, i)
        args = (fmt, x, F.cuda(wp), F.cuda(wt), F.cuda(wr))
        jobs.append((args, ops().linear_fp4_from_16bit(*args)))
    torch.cuda.synchronize()
    bad = []

    def work(args, want):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs = [ops().linear_fp4_from_16bit(*args) for _ in range(50)]
        s.synchronize()
        if not all(torch.equal(o, want) for o in outs):
            bad.append(args[0])
    threads = [threading.Thread(target=work, args=j) for j in jobs for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad
    import ctypes
    import duqlinear4bitcuda_b200.lib as L
    status = ctypes.c_int32(-1)
    L.call("duq4_last_device_status", L.current_stream(), ctypes.byref(status))
    assert status.value == 0


def test_captured_products_replay_side_by_side():
    """Two graphs of from_16bit, one with columns left over behind whole rounds, replayed at once on two streams."""
    made = []
    for fmt, m, n, k in (("nvfp4", 300, 9600, 1056), ("mxfp4", 20, 3000, 2048)):
        x = make(m, k, torch.float16, m).cuda()
        wp, wt, wr, _ = F.random_operand(fmt, n, k, 3)
        args = (fmt, x, F.cuda(wp), F.cuda(wt), F.cuda(wr) * 1e-4)
        want = ops().linear_fp4_from_16bit(*args)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops().linear_fp4_from_16bit(*args)
            out2 = ops().linear_fp4_from_16bit(*args)
        made.append((g, out, out2, want, torch.cuda.Stream(), args))
    for _ in range(5):
        for g, out, out2, want, s, _ in made:
            with torch.cuda.stream(s):
                out.zero_()
                g.replay()
    torch.cuda.synchronize()
    for g, out, out2, want, s, _ in made:
        assert torch.equal(out, want) and torch.equal(out2, want)


def test_offsets_beyond_32_bits():
    """More than 2^32 elements: the last rows of a quantizer, of a product's activations and of its result."""
    rows, cols = 66000, 65536
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x.view(torch.int16).random_(0x3F00, 0x4080)
    for fmt in FORMATS:
        codes, tiled, row = ops().fp4_quantize(fmt, x)
        some = ops().fp4_quantize(fmt, x[-128 - rows % 128:].contiguous())
        assert torch.equal(codes[-128 - rows % 128:], some[0])
        tail = tiled[-some[1].numel():]
        blocks = cols // F.BLOCK[fmt]
        assert np.array_equal(F.untile(tail.cpu().numpy(), 128 + rows % 128, blocks), F.untile(some[1].cpu().numpy(), 128 + rows % 128, blocks))
        assert row is None or torch.equal(row[-200:], some[2][-200:])
        back = ops().fp4_dequantize(fmt, codes, tiled, row, torch.bfloat16)
        assert torch.equal(back[-100:], ops().fp4_dequantize(fmt, *some, torch.bfloat16)[-100:])
        del back
        wp, wt, wr, _ = F.random_operand(fmt, 40, cols, 3)
        w = (F.cuda(wp), F.cuda(wt), F.cuda(wr))
        y = ops().linear_fp4(fmt, codes, tiled, row, *w, None, torch.bfloat16)
        few = ops().linear_fp4(fmt, *some, *w, None, torch.bfloat16)
        assert torch.allclose(y[-200:].float(), few[-200:].float(), rtol=2 ** -6, atol=1e-2 * few.float().abs().max().item())
        del codes, tiled, row, y
    del x
    m, n, k = 70000, 65536, 64
    ap, at, ar, av = F.random_operand("nvfp4", m, k, 1)
    wp, wt, wr, wv = F.random_operand("nvfp4", n, k, 2)
    y = ops().linear_fp4("nvfp4", F.cuda(ap), F.cuda(at), F.cuda(ar), F.cuda(wp), F.cuda(wt), F.cuda(wr), None, torch.bfloat16)
    for r in (0, 65535, 65536, m - 1):
        check_product(y[r:r + 1], av[r:r + 1], wv, None, torch.bfloat16)


@pytest.mark.parametrize("fmt", FORMATS)
def test_refusals_on_the_gpu(fmt):
    """Wrong sizes, layouts and alignments of tensors that are on the GPU raise and launch nothing."""
    o = ops()
    x = make(8, 128, torch.float16).cuda()
    q = o.fp4_quantize(fmt, x)
    w = torch.ones(128, dtype=torch.float16, device="cuda")
    for call, match in [
        (lambda: o.fp4_quantize(fmt, x[:, :100].contiguous()), "multiple of 32"),
        (lambda: o.fp4_quantize(fmt, x.t()), "contiguous"),
        (lambda: o.fp4_quantize(fmt, torch.empty(4, 65568, dtype=torch.float16, device="cuda")), "shape"),
        (lambda: o.fp4_quantize(fmt, x.view(-1)[4:4 + 256].view(2, 128)), "aligned"),
        (lambda: o.fp4_dequantize(fmt, q[0], q[1][:-1], q[2], torch.float16), "bytes"),
        (lambda: o.fp4_dequantize("nvfp4", q[0], q[1] if fmt == "nvfp4" else o.fp4_quantize("nvfp4", x)[1], None, torch.float16), "row_scales"),
        (lambda: o.linear_fp4(fmt, *q, q[0][:, :32].contiguous(), q[1], q[2]), "bytes|disagree"),
        (lambda: o.linear_fp4(fmt, *q, *q, torch.ones(7, dtype=torch.float16, device="cuda")), "bias to have 8 entries"),
        (lambda: o.linear_fp4_from_16bit(fmt, x[:, :64].contiguous(), *q), "disagree on K"),
        (lambda: o.norm_residual_quantize(fmt, x, w[:64]), "weight to have 128"),
        (lambda: o.norm_residual_quantize(fmt, x, w, post_weight=w), "go with residual"),
        (lambda: o.norm_residual_quantize(fmt, x, w, residual=x[:4]), "disagree on their shape"),
        (lambda: o.norm_residual_quantize(fmt, x, w, residual=x, gate=x[:4]), "gate must be"),
        (lambda: o.norm_residual_quantize(fmt, x, w, -1.0), "eps"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            call()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 22016, 4096), (1, 4096, 11008), (16, 4096, 4096), (2, 129, 32), (16, 40, 96), (7, 300, 2080), (3, 1000, 4128),
                                   (13, 20000, 1056), (1, 100, 65536), (5, 513, 8192)])
def test_few_tokens_from_16bit(fmt, dtype, m, n, k):
    """Few tokens on long and short layers equal quantizer and product, bit for bit; bad tokens and zero tokens among them."""
    x = make(m, k, dtype, m + k).cuda()
    if m > 4:
        x[1] = 0
        x[2, k - 1] = float("inf")
        x[3, 0] = float("nan")
    wp, wt, wr, _ = F.random_operand(fmt, n, k, 11)
    w = (F.cuda(wp), F.cuda(wt), F.cuda(wr))
    bias = make(1, n, dtype, 9)[0].cuda()
    want = ops().linear_fp4(fmt, *ops().fp4_quantize(fmt, x), *w, bias, dtype)
    got = ops().linear_fp4_from_16bit(fmt, x, *w, bias)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("fmt", ["sym", "asym"])
@pytest.mark.parametrize("rows,cols", [(2, 65536), (400, 32), (700, 512), (1200, 11008)])
def test_norm_into_the_integer_layers(fmt, rows, cols):
    """The integer formats at the widest and the narrowest rows, and on into the layer that takes them."""
    import duqlinear4bitcuda_b200.nn as nn
    x, residual = make(rows, cols, torch.float16, 1).cuda(), make(rows, cols, torch.float16, 2).cuda()
    joint = nn.NormResidualQuantizer(cols, fmt, eps=1e-5, post_norm=True, residual_scale=0.5).cuda()
    q, stream = joint(x, residual)
    r, h = _joint(x, joint.weight, 1e-5, residual, joint.post_weight, None, 0.5)
    assert torch.equal(stream, r)
    want = (nn.SymQuantizer() if fmt == "sym" else nn.AsymQuantizer())(h)
    assert torch.equal(q.quantized_x, want.quantized_x) and torch.equal(q.scales_x.flatten(), want.scales_x.flatten())
    if fmt == "asym":
        assert torch.equal(q.zeros_x.flatten(), want.zeros_x.flatten())
    elif cols % 64 == 0:
        lin = nn.Linear4bitSQ(cols, 64).cuda()
        lin.weight_scales.fill_(0.01)
        assert torch.equal(lin(q), lin(want))


@pytest.mark.parametrize("static", [0, 1])
@pytest.mark.parametrize("fmt", FORMATS)
def test_a_long_chain_of_launches_keeps_its_order(fmt, static):
    """Launches that overlap the ones in front: a chain in which every call reads what the call before wrote, buffers reused all the
    time, integer layers and plain torch kernels between; with and without the promise on weights. As the same chain with a
    wait after every call."""
    import duqlinear4bitcuda_b200.lib as L
    import duqlinear4bitcuda_b200.nn as nn
    g = torch.Generator().manual_seed(1)
    dim, dtype = 512, torch.float16
    lin = lambda i, o: torch.nn.Linear(i, o, bias=True).to(dtype).cuda()
    up, down = nn.LinearFP4.from_linear(lin(dim, 2 * dim), fmt, dtype), nn.LinearFP4.from_linear(lin(dim, dim), fmt, dtype)
    tall = nn.LinearFP4.from_linear(lin(dim, 20000), fmt, dtype)
    integer = nn.Linear4bitASQ(dim, dim).cuda()
    integer.weight_scales.fill_(0.05)
    joint, glue = nn.NormResidualQuantizer(dim, fmt, post_norm=True, residual_scale=0.5, dtype=dtype).cuda(), nn.SiluMulQuantizerFP4(fmt)

    def chain(x, wait):
        stream = x
        for i in range(12):
            for f in ((lambda t: up(t)), (lambda t: glue(t)), (lambda t: down(t))):
                x = f(x)
                if wait:
                    torch.cuda.synchronize()
            q, stream = joint(x, stream)
            x = q.dequantize(dtype)
            if wait:
                torch.cuda.synchronize()
            x = integer(x) * 0.5 if i % 3 == 0 else x + 0.25
            if i % 4 == 0:
                x = x + tall(x)[:, 7:7 + dim] * 0.1
            if wait:
                torch.cuda.synchronize()
            x = x.clamp(-8, 8)
        return x, stream
    old = L.cdll.duq4_set_static_weights(static)
    try:
        for tokens in (1, 17, 140, 700):
            x = torch.randn(tokens, dim, generator=g).to(dtype).cuda()
            want = chain(x, True)
            for _ in range(3):
                got = chain(x, False)
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    finally:
        L.cdll.duq4_set_static_weights(old)
