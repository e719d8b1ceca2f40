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
