"""(new) Modules of the microscaled 4-bit formats, siblings of the integer quantizers and linear layers; the reference has
none of this kind. `format` is "mxfp4" (a power-of-two scale per 32 neighbours) or "nvfp4" (an e4m3 scale per 16 and a float
per row)."""
import torch

from .. import _CUDA as ops
from ..tools import quantization as qz
from ..tools.tensor_utils import PackedFP4Tensor, PackedQuantizedTensor
from .quantizer import _as_rows, _scale_shape


def _check_format(format):
    if format not in qz.FP4_BLOCK:
        raise ValueError(f"unknown format {format!r} (mxfp4, nvfp4)")
    return format


def _packed(format, parts, lead, dtype):
    codes, block_scales, row_scales = parts
    return PackedFP4Tensor(format, codes.view(*lead, codes.shape[1]), block_scales, row_scales, dtype)


class QuantizerFP4(torch.nn.Module):
    """fp16 / bfloat16 [..., K] -> PackedFP4Tensor in one kernel. K % 32 == 0."""

    def __init__(self, format="nvfp4"):
        super().__init__()
        self.format = _check_format(format)

    def forward(self, x) -> PackedFP4Tensor:
        x2, lead = _as_rows(x)
        return _packed(self.format, ops.fp4_quantize(self.format, x2), lead, x.dtype)


class SiluMulQuantizerFP4(torch.nn.Module):
    """[..., 2*I], gate projection first -> the PackedFP4Tensor of F.silu(gate) * up, which is not stored."""

    def __init__(self, format="nvfp4"):
        super().__init__()
        self.format = _check_format(format)

    def forward(self, gate_up) -> PackedFP4Tensor:
        x2, lead = _as_rows(gate_up)
        return _packed(self.format, ops.fp4_silu_mul_quantize(self.format, x2), lead, gate_up.dtype)


def _rows_of(name, t, x, rows, broadcast):
    """t as the rows [rows, C] of x: of x's shape but for leading ones, flattened already, or (a gate) whatever broadcasts to
    x's shape. As many rows in another arrangement are refused: they would meet the wrong tokens."""
    while t.dim() > x.dim() and t.shape[0] == 1:
        t = t[0]
    if t.shape == x.shape or t.shape == (rows, x.shape[-1]):
        return _as_rows(t)[0]
    if t.dim() > x.dim() or any(a not in (1, b) for a, b in zip(t.shape[::-1], x.shape[::-1])) or not (broadcast or t.numel() == x.numel()):
        raise ValueError(f"{name} of shape {tuple(t.shape)} does not go with x of shape {tuple(x.shape)}")
    return _as_rows(t.expand(x.shape))[0]


class NormResidualQuantizer(torch.nn.Module):
    """The joint between two blocks of a transformer in one kernel: the norm after a block (post_norm=True), its gate and
    residual scale, the residual sum, the norm before the next block, and the quantizer in front of its first layer.

        forward(x)                  -> quantized norm(x) * weight
        forward(x, residual, gate)  -> (quantized norm(r) * weight, r),
                                       r = residual + residual_scale * gate * [norm(x) * post_weight]

    norm(t) = t / sqrt(mean(t^2) + eps) over the last dimension. residual: like x. gate: None, [dim], or what broadcasts to x
    (one per sequence, [B, 1, dim], is copied to one per token). format: "mxfp4" / "nvfp4" (a PackedFP4Tensor for
    LinearFP4), "sym" / "asym" (a PackedQuantizedTensor for the integer layers, fp16), "none" (the norm itself).
    input_clip_ratio: as SymQuantizer's, for "sym" only. dim % 32 == 0."""

    def __init__(self, dim, format="nvfp4", eps=1e-6, post_norm=False, residual_scale=1.0, dtype=torch.float16, input_clip_ratio=1.0):
        super().__init__()
        if format not in ("none", "sym", "asym"):
            _check_format(format)
        self.format, self.eps, self.residual_scale, self.input_clip_ratio = format, eps, residual_scale, input_clip_ratio
        self.register_buffer("weight", torch.ones(dim, dtype=dtype))
        if post_norm:
            self.register_buffer("post_weight", torch.ones(dim, dtype=dtype))
        else:
            self.post_weight = None

    def forward(self, x, residual=None, gate=None):
        x2, lead = _as_rows(x)
        post = None
        if residual is not None:
            residual = _rows_of("residual", residual, x, x2.shape[0], False)
            post = self.post_weight
            if gate is not None and gate.dim() > 1 and gate.numel() == gate.shape[-1]:
                gate = gate.reshape(-1)   # one for all tokens
            if gate is not None and gate.shape != x.shape[-1:]:
                gate = _rows_of("gate", gate, x, x2.shape[0], True)
        stream, *q = ops.norm_residual_quantize(self.format, x2, self.weight, self.eps, residual, post, gate, self.residual_scale,
                                               self.input_clip_ratio)
        if self.format == "none":
            out = q[0].view(x.shape)
        elif self.format == "sym":
            out = PackedQuantizedTensor(q[0].view(*lead, q[0].shape[1]), q[1].view(_scale_shape(lead)))
        elif self.format == "asym":
            out = PackedQuantizedTensor(q[0].view(*lead, q[0].shape[1]), q[1].view(*lead, 1), q[2].view(*lead, 1))
        else:
            out = _packed(self.format, q, lead, x.dtype)
        return out if residual is None else (out, stream.view(x.shape))


class LinearFP4(torch.nn.Module):
    """Linear layer on microscaled 4-bit weights and activations. Buffers: weight uint8 [out, in/2], weight_scales uint8
    (block scales in the tensor cores' tile order; qz.fp4_tile_scales makes it from [out, in/block]), weight_row_scales
    float [out] (the nvfp4 format's second scale; a checkpoint's one float per tensor is that float in every row), bias.
    forward takes 16-bit activations (quantized on the way, the result has their type) or a PackedFP4Tensor; a bias of another
    type than theirs is rounded to it in every call."""

    def __init__(self, in_features, out_features, bias=False, format="nvfp4", dtype=torch.float16):
        super().__init__()
        if in_features % 32 != 0:
            raise ValueError("in_features must be a multiple of 32")
        self.in_features, self.out_features, self.format = in_features, out_features, _check_format(format)
        blocks = in_features // qz.FP4_BLOCK[format]
        self.register_buffer("weight", torch.zeros((out_features, in_features // 2), dtype=torch.uint8))
        self.register_buffer("weight_scales", torch.zeros(-(-out_features // 128) * -(-blocks // 4) * 512, dtype=torch.uint8))
        if format == "nvfp4":
            self.register_buffer("weight_row_scales", torch.ones(out_features, dtype=torch.float32))
        else:
            self.weight_row_scales = None
        if bias:
            self.register_buffer("bias", torch.zeros(out_features, dtype=dtype))
        else:
            self.bias = None

    def _apply(self, fn, recurse=True):
        # .half(), .to(dtype) and the like convert every floating-point buffer of a model; the row scales are part of the
        # format, 32 bits whatever the layer's type, and only follow the device
        rows = self.weight_row_scales
        super()._apply(fn, recurse)
        if rows is not None and self.weight_row_scales.dtype != torch.float32:
            self.weight_row_scales = rows.to(self.weight_row_scales.device)
        return self

    def _bias_as(self, dtype):
        return self.bias if self.bias is None or self.bias.dtype == dtype else self.bias.to(dtype)

    def forward(self, x):
        w = (self.weight, self.weight_scales, self.weight_row_scales)
        if isinstance(x, PackedFP4Tensor):
            if x.format != self.format:
                raise ValueError(f"activations are {x.format}, the weights {self.format}")
            codes, lead = _as_rows(x.codes)
            y = ops.linear_fp4(self.format, codes, x.block_scales, x.row_scales, *w, self._bias_as(x.dtype), x.dtype)
        else:
            x2, lead = _as_rows(x)
            y = ops.linear_fp4_from_16bit(self.format, x2, *w, self._bias_as(x.dtype))
        return y.view(*lead, self.out_features)

    @classmethod
    def from_linear(cls, module: torch.nn.Linear, format="nvfp4", dtype=None):
        """Quantizes the weights of a Linear on the GPU; the buffers stay there. dtype: of the bias, that is of the
        activations the layer will see; the module's own where that has 16 bits, else fp16."""
        if dtype is None:
            dtype = module.weight.dtype if module.weight.dtype in (torch.float16, torch.bfloat16) else torch.float16
        new = cls(module.in_features, module.out_features, module.bias is not None, format, dtype)
        w = module.weight.data
        if w.dtype not in (torch.float16, torch.bfloat16):
            w = w.to(dtype)
        new = new.to(w.device if w.is_cuda else "cuda")
        codes, scales, rows = ops.fp4_quantize(format, w.to(new.weight.device).contiguous())
        new.weight.copy_(codes)
        new.weight_scales.copy_(scales)
        if rows is not None:
            new.weight_row_scales.copy_(rows)
        if module.bias is not None:
            new.bias.copy_(module.bias.detach())
        return new
