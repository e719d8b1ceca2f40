"""Modules of the fp4 operators as a model uses them: types of a layer and of its activations."""
import pytest
import torch

pytestmark = pytest.mark.gpu
H, B = torch.float16, torch.bfloat16


def layer(dtype):
    torch.manual_seed(3)
    return torch.nn.Linear(128, 72, bias=True).to(dtype).cuda()


def product(q, x, bias):
    """The operator itself on the layer's weights, with a bias of the activations' type."""
    import duqlinear4bitcuda_b200._CUDA as o
    return o.linear_fp4_from_16bit(q.format, x, q.weight, q.weight_scales, q.weight_row_scales, bias)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("own", [H, B])
def test_a_layer_takes_its_own_activations(fmt, own):
    """from_linear keeps the type of a 16-bit layer, so that what the layer took the new one takes."""
    import duqlinear4bitcuda_b200.nn as nn
    lin = layer(own)
    q = nn.LinearFP4.from_linear(lin, fmt)
    assert q.bias.dtype == own and torch.equal(q.bias, lin.bias)
    x = torch.randn(5, 128, device="cuda").to(own)
    y = q(x)
    assert y.dtype == own and torch.equal(y, product(q, x, lin.bias.detach()))
    assert torch.equal(q(nn.QuantizerFP4(fmt)(x)), y)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("own,given,acts", [(torch.float32, None, H), (torch.float32, B, B), (B, H, H), (H, B, B),
                                            (B, None, H), (H, None, B), (torch.float32, None, B)])
def test_a_bias_of_another_type_is_rounded_to_the_activations(fmt, own, given, acts):
    import duqlinear4bitcuda_b200.nn as nn
    lin = layer(own)
    q = nn.LinearFP4.from_linear(lin, fmt) if given is None else nn.LinearFP4.from_linear(lin, fmt, given)
    kept = given or (own if own in (H, B) else H)
    assert q.bias.dtype == kept
    x = torch.randn(3, 128, device="cuda").to(acts)
    want = product(q, x, lin.bias.detach().to(kept).to(acts))
    assert torch.equal(q(x), want) and torch.equal(q(nn.QuantizerFP4(fmt)(x)), want)
    assert torch.equal(q.float()(x), want)      # a bias that a conversion of the model left in 32 bits


@pytest.mark.parametrize("ratio", [1.0, 0.8])
def test_joint_with_a_clip_ratio_equals_the_quantizer(ratio):
    import duqlinear4bitcuda_b200.nn as nn
    x, r = torch.randn(7, 96, device="cuda").half(), torch.randn(7, 96, device="cuda").half()
    h, _ = nn.NormResidualQuantizer(96, "none").cuda()(x, r)
    got, _ = nn.NormResidualQuantizer(96, "sym", input_clip_ratio=ratio).cuda()(x, r)
    want = nn.SymQuantizer(ratio)(h)
    assert torch.equal(got.quantized_x, want.quantized_x) and torch.equal(got.scales_x, want.scales_x)


@pytest.mark.parametrize("shape", [(128,), (1, 1, 128), (4, 1, 128), (1, 5, 128), (4, 5, 128), (20, 128)])
def test_joint_with_gates_that_broadcast(shape):
    """A gate per channel, sequence, position and token equals the same gate written out for every token."""
    import duqlinear4bitcuda_b200.nn as nn
    x, r, g = torch.randn(4, 5, 128, device="cuda").to(B), torch.randn(4, 5, 128, device="cuda").to(B), torch.randn(shape, device="cuda").to(B)
    joint = nn.NormResidualQuantizer(128, "nvfp4", post_norm=True, dtype=B).cuda()
    q, stream = joint(x, r, g)
    full = (g.view(4, 5, 128) if shape == (20, 128) else g.expand(4, 5, 128)).contiguous()
    want, wstream = joint(x, r, full)
    assert torch.equal(q.codes, want.codes) and torch.equal(stream, wstream) and torch.equal(q.dequantize(), want.dequantize())
