"""Microscaled 4-bit floating-point operators (mxfp4, nvfp4): what they compute, on which sizes they are measured.

Formats. An element is an e2m1 number (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives; round to nearest, ties to the even
code, saturating at 6). "mxfp4" keeps one power-of-two scale per 32 neighbours of a row, 2^(floor(log2 max|x|) - 2); "nvfp4"
one e4m3 scale per 16 neighbours and one float per row: the row's scale is max|row| / 2688 rounded to 8 bits (bfloat16; not
below 2^-110), the block's e4m3(max|block| / (6 * row scale)). With 8 bits the product of the two scales is exact, and no
quotient of a 16-bit value by it comes so near to the middle of two codes, without being it, that 32 bits could not tell.

Operators: "quantize" (and reading back), "silu" (silu(gate) * up quantized without being stored), "norm" (root-mean-square
norms around a residual sum with a gate and a scale, the second norm's result quantized) and "linear" (16-bit activations,
quantized per token, times 4-bit weights).
"""
import math

import torch

own = False

FORMATS = ("mxfp4", "nvfp4")
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def listed():
    return [
        # one token of a 4096-wide layer being decoded: latency
        {"name": "quantize-nv-1x4096", "op": "quantize", "format": "nvfp4", "dtype": "f16", "rows": 1, "cols": 4096},
        # the activations of a 4096-token prompt in front of the 8192-wide layer
        {"name": "quantize-mx-4096x8192", "op": "quantize", "format": "mxfp4", "dtype": "bf16", "rows": 4096, "cols": 8192},
        # gate and up projections of an 11008-wide MLP: 16 sequences being decoded, and a batch of prompts
        {"name": "silu-nv-16x11008", "op": "silu", "format": "nvfp4", "dtype": "f16", "rows": 16, "cols": 11008},
        {"name": "silu-mx-16384x11008", "op": "silu", "format": "mxfp4", "dtype": "f16", "rows": 16384, "cols": 11008},
        # the joint between two blocks: one token; a ragged prompt with a gate per token and no norm after the block;
        # a long prompt with all parts
        {"name": "norm-nv-1x4096", "op": "norm", "format": "nvfp4", "dtype": "f16", "rows": 1, "cols": 4096, "post": True, "gate": "none"},
        {"name": "norm-nv-1001x4096", "op": "norm", "format": "nvfp4", "dtype": "f16", "rows": 1001, "cols": 4096, "post": False, "gate": "row"},
        {"name": "norm-mx-4096x8192", "op": "norm", "format": "mxfp4", "dtype": "bf16", "rows": 4096, "cols": 8192, "post": True, "gate": "channel"},
        # the fused gate/up layer for one token, a square layer for 16, a down projection with a bias for an odd batch,
        # and the wide layer for a short and for a long prompt
        {"name": "linear-nv-1-4096-22016", "op": "linear", "format": "nvfp4", "dtype": "f16", "rows": 1, "cols": 4096, "out": 22016, "bias": False},
        {"name": "linear-mx-16-4096-4096", "op": "linear", "format": "mxfp4", "dtype": "f16", "rows": 16, "cols": 4096, "out": 4096, "bias": False},
        {"name": "linear-nv-77-11008-4096", "op": "linear", "format": "nvfp4", "dtype": "bf16", "rows": 77, "cols": 11008, "out": 4096, "bias": True},
        {"name": "linear-mx-512-8192-28672", "op": "linear", "format": "mxfp4", "dtype": "f16", "rows": 512, "cols": 8192, "out": 28672, "bias": False},
        {"name": "linear-nv-4096-8192-28672", "op": "linear", "format": "nvfp4", "dtype": "bf16", "rows": 4096, "cols": 8192, "out": 28672, "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("quantize", "silu", "norm", "linear", "linear", "linear"))
    case = {"op": op, "format": rng.choice(FORMATS), "dtype": rng.choice(("f16", "bf16"))}
    if op == "linear":
        case["cols"] = 32 * _log(rng, 2, 896)
        case["out"] = _log(rng, 33, 28672)
        case["rows"] = _log(rng, 1, min(16384, (4096 * 8192 * 28672) // (case["cols"] * case["out"])))
        case["bias"] = rng.random() < 0.5
        return case
    case["cols"] = 32 * _log(rng, 2, 896)
    case["rows"] = _log(rng, 1, min(16384, (4096 * 8192) // case["cols"]))
    if op == "norm":
        case["post"] = rng.random() < 0.5
        case["gate"] = rng.choice(("none", "channel", "row"))
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(gen, rows, cols, dt):
    """Tokens as layers see them: about normal, a few loud channels; of many, the last ones are padding (zeros)."""
    x = _normal(gen, rows, cols)
    loud = torch.rand(cols, generator=gen, device="cuda") < 0.005
    x = x * torch.where(loud, 20.0, 1.0)
    if rows >= 64:
        x[rows - rows // 64:] = 0
    return x.to(dt)


def _tiled(scales):
    """Row-major block scales [rows, blocks] as the operators keep them: tiles of 128 rows x 4 blocks, 512 bytes each, in
    which row r holds its four bytes at 16 * (r % 32) + 4 * (r // 32)."""
    rows, blocks = scales.shape
    tr, tb = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros(tr * 128, tb * 4, dtype=torch.uint8, device=scales.device)
    full[:rows, :blocks] = scales
    return full.view(tr, 4, 32, tb, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, rows, cols, fmt = DTYPES[case["dtype"]], case["rows"], case["cols"], case["format"]
    s = {"op": case["op"], "format": fmt, "dtype": dt}
    if case["op"] == "quantize":
        s["x"] = _activations(gen, rows, cols, dt)
    elif case["op"] == "silu":
        s["gate_up"] = (_normal(gen, rows, 2 * cols) * 1.5).to(dt)
    elif case["op"] == "norm":
        s["x"] = _activations(gen, rows, cols, dt)
        s["residual"] = (_activations(gen, rows, cols, dt).float() * 3).to(dt)
        s["weight"] = (1 + 0.1 * _normal(gen, cols)).to(dt)
        s["post_weight"] = (0.5 + 0.1 * _normal(gen, cols)).to(dt) if case["post"] else None
        s["gate"] = None if case["gate"] == "none" else (0.7 * _normal(gen, *((rows,) if case["gate"] == "row" else ()), cols)).to(dt)
        s["eps"], s["residual_scale"] = 1e-5, 0.25
    else:
        n = case["out"]
        s["x"] = _activations(gen, rows, cols, dt)
        # weights as a checkpoint holds them: codes and block scales, made once; the tiled copy of the scales is kept beside
        s["w"] = torch.randint(0, 256, (n, cols // 2), generator=gen, device="cuda", dtype=torch.uint8)
        if fmt == "mxfp4":
            s["w_scales"] = torch.randint(116, 120, (n, cols // 32), generator=gen, device="cuda", dtype=torch.uint8)
            s["w_rows"] = None
        else:
            s["w_scales"] = torch.randint(0x50, 0x7F, (n, cols // 16), generator=gen, device="cuda", dtype=torch.uint8)
            s["w_rows"] = (0.5 + torch.rand(n, generator=gen, device="cuda")) * (2.0 / 448 / math.sqrt(cols) / 6)
        s["w_tiled"] = _tiled(s["w_scales"])
        s["bias"] = _normal(gen, n).to(dt) if case["bias"] else None
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------

def _e2m1(x):
    """x (float) rounded to e2m1: below 2 in halves, below 4 in ones, above in twos; torch.round takes ties to the even."""
    a = x.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.round(a / step) * step * torch.where(x < 0, -1.0, 1.0)


def _power(e):
    """2^e as a float, for whole e in [-126, 127], made of its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _round_trip(h, fmt):
    """h [rows, cols] -> the values its 4-bit form stands for, float."""
    rows, cols = h.shape
    x = h.float().view(rows, cols // BLOCK[fmt], BLOCK[fmt])
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        e = torch.where(top > 0, torch.frexp(top).exponent - 3, -126).clamp(min=-126)
        v = _e2m1(x * _power(-e)) * _power(e)
    else:
        row = (top.amax(1, keepdim=True) / 2688.0).bfloat16().float().clamp(min=2.0 ** -110)
        block = (top / (6.0 * row)).to(torch.float8_e4m3fn).float()
        d = block * row
        v = torch.where(block > 0, _e2m1(x / torch.where(block > 0, d, 1.0)), 0.0) * d
    return v.view(rows, cols)


def _rms(x, eps):
    """1 / root mean square of each row. The sum is taken in 64 bits: the codes behind it jump at borders."""
    x = x.double()
    return (1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)).float()


_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _weights(s):
    """The weights as floats [out, cols]."""
    table = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device="cuda")
    w = s["w"]
    v = table[torch.stack((w & 15, w >> 4), -1).view(w.shape[0], -1).int()]
    if s["format"] == "mxfp4":
        scale = _power(s["w_scales"].int() - 127)
    else:
        scale = s["w_scales"].view(torch.float8_e4m3fn).float() * s["w_rows"][:, None]
    return (v.view(*scale.shape, -1) * scale[..., None]).view(v.shape)


def _silu(g):
    return g / (1.0 + torch.exp(-g))


def _plain(s):
    dt, fmt = s["dtype"], s["format"]
    if s["op"] == "quantize":
        return {"values": _round_trip(s["x"], fmt).to(dt)}
    if s["op"] == "silu":
        gate, up = s["gate_up"].float().chunk(2, -1)
        h = (_silu(gate).to(dt).float() * up).to(dt)   # the two roundings of silu(gate) * up on 16-bit tensors
        return {"values": _round_trip(h, fmt).to(dt)}
    if s["op"] == "norm":
        y = s["x"].float()
        if s["post_weight"] is not None:
            y = y * _rms(y, s["eps"]) * s["post_weight"].float()
        if s["gate"] is not None:
            y = y * s["gate"].float()
        r = (s["residual"].float() + y * s["residual_scale"]).to(dt)   # the stream is kept in 16 bits; the norm reads it
        h = (r.float() * _rms(r, s["eps"]) * s["weight"].float()).to(dt)
        return {"residual": r, "values": _round_trip(h, fmt).to(dt)}
    y = _round_trip(s["x"], fmt) @ _weights(s).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return {"y": y.to(dt)}


def _own(s):
    from duqlinear4bitcuda_b200 import _CUDA as ops
    dt, fmt = s["dtype"], s["format"]
    if s["op"] == "quantize":
        return {"values": ops.fp4_dequantize(fmt, *ops.fp4_quantize(fmt, s["x"]), dt)}
    if s["op"] == "silu":
        return {"values": ops.fp4_dequantize(fmt, *ops.fp4_silu_mul_quantize(fmt, s["gate_up"]), dt)}
    if s["op"] == "norm":
        residual, *quantized = ops.norm_residual_quantize(fmt, s["x"], s["weight"], s["eps"], s["residual"], s["post_weight"], s["gate"],
                                                          s["residual_scale"])
        return {"residual": residual, "values": ops.fp4_dequantize(fmt, *quantized, dt)}
    return {"y": ops.linear_fp4_from_16bit(fmt, s["x"], s["w"], s["w_tiled"], s["w_rows"], s["bias"])}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------

def work(case):
    rows, cols, block = case["rows"], case["cols"], BLOCK[case["format"]]
    n = rows * cols
    coded = n // 2 + n // block + (4 * rows if block == 16 else 0)   # codes, block scales, row scales
    if case["op"] == "quantize":
        return {"bytes": 2 * n + 2 * coded + 2 * n, "flops": 6 * n}       # read, coded form out and in again, values out
    if case["op"] == "silu":
        return {"bytes": 4 * n + 2 * coded + 2 * n, "flops": 12 * n}
    if case["op"] == "norm":
        gate = {"none": 0, "channel": 2 * cols, "row": 2 * n}[case["gate"]]
        return {"bytes": 4 * n + gate + 4 * cols + 2 * n + 2 * coded + 2 * n, "flops": 16 * n}
    out = case["out"]
    weights = out * cols // 2 + out * cols // block + (4 * out if block == 16 else 0)
    return {"bytes": 2 * n + weights + 2 * rows * out + (2 * out if case["bias"] else 0), "flops": 2 * n * out}


# ---- from the definitions, in 64 bits -------------------------------------------------------------------------------

def _grid(signed, limit):
    """The values of a small float format, ascending: e2m1 ("limit" 6) or positive e4m3 (448)."""
    if limit == 6:
        return torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device="cuda")
    steps = [m * 2.0 ** -9 for m in range(8)]
    steps += [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    return torch.tensor(steps[:127], dtype=torch.float64, device="cuda")


def _nearest(a, grid):
    """The nearest value of the grid to each a >= 0; of two equally near, the one with the even index."""
    up = torch.searchsorted(grid, a.contiguous()).clamp(1, grid.numel() - 1)
    lo, hi = grid[up - 1], grid[up]
    middle = (lo + hi) / 2
    take = (a > middle) | ((a == middle) & (up % 2 == 0))
    return torch.where(take, hi, lo)


def _exact_round_trip(h, fmt):
    rows, cols = h.shape
    out = torch.empty(rows, cols, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 2048):
        x = h[at:at + 2048].double().reshape(-1, cols // BLOCK[fmt], BLOCK[fmt])
        top = x.abs().amax(-1, keepdim=True)
        if fmt == "mxfp4":
            t = torch.where(top > 0, top, 1.0)
            e = torch.floor(torch.log2(t))   # the logarithm of a power of two may come out below it
            e = e + (torch.exp2(e + 1) <= t).double() - (torch.exp2(e) > t).double()
            scale = torch.exp2(e - 2)
        else:
            row = top.amax(1, keepdim=True) / 2688
            step = torch.exp2(torch.floor(torch.log2(torch.where(row > 0, row, 1.0))) - 7)
            row = torch.round(row / step) * step   # 8 bits
            scale = _nearest(top / (6 * torch.where(row > 0, row, 1.0)), _grid(False, 448)) * row
        q = _nearest(x.abs() / torch.where(scale > 0, scale, 1.0), _grid(True, 6))
        out[at:at + 2048] = (q * torch.sign(x) * scale).reshape(-1, cols)
    return out


def _exact_weights(s):
    w = s["w"].long()
    codes = torch.empty(w.shape[0], 2 * w.shape[1], dtype=torch.int64, device="cuda")
    codes[:, 0::2], codes[:, 1::2] = w % 16, w // 16
    v = _grid(True, 6)[codes % 8] * (1 - 2 * (codes // 8)).double()
    if s["format"] == "mxfp4":
        scale = torch.exp2(s["w_scales"].double() - 127)
    else:
        scale = _grid(False, 448)[s["w_scales"].long()] * s["w_rows"].double()[:, None]
    return v * scale.repeat_interleave(BLOCK[s["format"]], 1)


def exact(case, seed):
    s = prepare(case, seed)
    fmt, dt = s["format"], s["dtype"]
    if s["op"] == "quantize":
        return {"values": _exact_round_trip(s["x"], fmt)}
    if s["op"] == "silu":
        g, u = s["gate_up"].chunk(2, -1)
        h = torch.empty_like(g)
        for at in range(0, g.shape[0], 2048):
            part = g[at:at + 2048].double()
            h[at:at + 2048] = ((part * torch.sigmoid(part)).to(dt).double() * u[at:at + 2048].double()).to(dt)
        return {"values": _exact_round_trip(h, fmt)}
    if s["op"] == "norm":
        def norm(t, w):
            return t * w.double() / torch.sqrt(t.square().mean(-1, keepdim=True) + s["eps"])
        branch = s["x"].double()
        if s["post_weight"] is not None:
            branch = norm(branch, s["post_weight"])
        if s["gate"] is not None:
            branch = branch * s["gate"].double()
        total = s["residual"].double() + s["residual_scale"] * branch
        h = norm(total.to(dt).double(), s["weight"]).to(dt)
        return {"residual": total, "values": _exact_round_trip(h, fmt)}
    x = _exact_round_trip(s["x"], fmt)
    y = x @ _exact_weights(s).T
    return {"y": y if s["bias"] is None else y + s["bias"].double()}
