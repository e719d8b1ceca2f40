"""CPU-only: what the fp4 modules do with types, shapes and options before any launch."""
import pytest
import torch

import duqlinear4bitcuda_b200.nn as nn

H, B = torch.float16, torch.bfloat16


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.to(B), lambda m: m.double(), lambda m: m.to(torch.device("cpu"), H),
                                     lambda m: torch.nn.Sequential(m).bfloat16()[0], lambda m: m.half().float().bfloat16()])
def test_row_scales_stay_float_when_the_model_is_converted(convert):
    """A loader converts a whole model at once; the nvfp4 format's row scales are 32-bit numbers and keep their bits."""
    m = nn.LinearFP4(64, 40, bias=True, format="nvfp4")
    rows = torch.rand(40) + 1e-6
    m.weight_row_scales.copy_(rows)
    m.weight.random_(0, 256)
    codes = m.weight.clone()
    m = convert(m)
    assert m.weight_row_scales.dtype == torch.float32 and torch.equal(m.weight_row_scales, rows)
    assert "weight_row_scales" in m.state_dict() and m.state_dict()["weight_row_scales"].dtype == torch.float32
    assert m.weight.dtype == torch.uint8 and torch.equal(m.weight, codes) and m.weight_scales.dtype == torch.uint8
    assert nn.LinearFP4(64, 40, format="mxfp4").half().weight_row_scales is None


def test_row_scales_follow_the_device():
    m = nn.LinearFP4(64, 40, format="nvfp4").to("meta")
    assert m.weight_row_scales.device.type == "meta" and m.weight_row_scales.dtype == torch.float32
    m = m.half().to_empty(device="cpu")
    assert m.weight_row_scales.device.type == "cpu" and m.weight_row_scales.dtype == torch.float32


class Recorder:
    """Stands in for the operator module: notes the call and gives back results of the right shapes."""

    def norm_residual_quantize(self, *args):
        self.args = args
        x, residual = args[1], args[4]
        rows, cols = x.shape
        return residual, torch.zeros(rows, cols // 2, dtype=torch.uint8), torch.zeros(rows, dtype=H), torch.zeros(rows, dtype=H)


@pytest.fixture
def recorder(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(nn.fp4, "ops", r)
    return r


@pytest.mark.parametrize("given,want", [({}, 1.0), ({"input_clip_ratio": 0.75}, 0.75)])
def test_clip_ratio_reaches_the_quantizer(recorder, given, want):
    """As SymQuantizer's."""
    q = nn.NormResidualQuantizer(64, "sym", **given)
    q(torch.zeros(3, 64, dtype=H))
    assert recorder.args[8] == want and q.input_clip_ratio == want


def joint(recorder, x, residual, gate=None):
    out, stream = nn.NormResidualQuantizer(64, "sym")(x, residual, gate)
    assert stream.shape == x.shape
    return recorder.args[4], recorder.args[6]


X = torch.arange(2 * 3 * 64).reshape(2, 3, 64).to(H)


@pytest.mark.parametrize("shape", [(3, 2, 64), (6, 1, 64), (2, 3, 32), (1, 3, 64), (64,), (5, 64)])
def test_residual_of_another_shape_is_refused(recorder, shape):
    """As many rows in another arrangement would pair tokens with tokens of other sequences."""
    with pytest.raises(ValueError, match="residual"):
        joint(recorder, X, torch.zeros(shape, dtype=H))


@pytest.mark.parametrize("shape", [(3, 2, 64), (6, 1, 64), (32,), (2, 64), (3, 1, 64), (2, 3, 1, 64), (5, 64)])
def test_gate_of_another_shape_is_refused(recorder, shape):
    with pytest.raises(ValueError, match="gate"):
        joint(recorder, X, X, torch.zeros(shape, dtype=H))


@pytest.mark.parametrize("x,shape", [(X, (2, 3, 64)), (X, (6, 64)), (X[:1], (3, 64)), (X[:1], (1, 3, 64)), (X[0], (1, 3, 64)), (X[0, 0], (64,)), (X[0, 0], (1, 1, 64))])
def test_residual_shapes(recorder, x, shape):
    r = torch.randn(shape).to(H)
    assert torch.equal(joint(recorder, x, r)[0], r.reshape(-1, 64))


@pytest.mark.parametrize("shape", [(64,), (1, 64), (1, 1, 64)])
def test_one_gate_for_all_tokens_is_handed_on_as_it_is(recorder, shape):
    g = torch.randn(shape).to(H)
    got = joint(recorder, X, X, g)[1]
    assert got.shape == (64,) and torch.equal(got, g.reshape(64)) and got.data_ptr() == g.data_ptr()


@pytest.mark.parametrize("shape", [(2, 3, 64), (6, 64), (2, 1, 64), (1, 3, 64), (3, 64)])
def test_gates_of_tokens_sequences_and_positions(recorder, shape):
    """Whatever broadcasts to x: a gate per token, per sequence, per position."""
    g = torch.randn(shape).to(H)
    got = joint(recorder, X, X, g)[1]
    want = g if shape == (6, 64) else (torch.ones(2, 3, 64, dtype=H) * g).reshape(6, 64)
    assert got.is_contiguous() and torch.equal(got, want)
