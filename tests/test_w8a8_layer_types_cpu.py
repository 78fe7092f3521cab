"""The type of an 8-bit layer when its model is cast, with and without a bias.  No GPU needed."""

import copy

import pytest
import torch

from nunchaku_amd.models import W8A8Linear


@pytest.mark.parametrize("bias", [True, False])
def test_the_layers_type_goes_with_the_model(bias):
    torch.manual_seed(0)
    m = W8A8Linear.from_linear(torch.nn.Linear(96, 40, bias=bias, dtype=torch.bfloat16))
    assert m.torch_dtype == torch.bfloat16
    scales = m.wscales.clone()
    model = torch.nn.Sequential(m)
    for cast, want in (
        (lambda t: t.half(), torch.float16), (lambda t: t.cpu(), torch.float16), (lambda t: t.to(torch.bfloat16), torch.bfloat16),
        (lambda t: t.to("cpu", torch.float16), torch.float16), (lambda t: t.float(), torch.float32), (lambda t: t.requires_grad_(False), torch.float32),
        (lambda t: t.bfloat16(), torch.bfloat16), (lambda t: copy.deepcopy(t), torch.bfloat16), (lambda t: t.share_memory(), torch.bfloat16),
    ):
        model = cast(model)
        assert model[0].torch_dtype == want
        assert model[0].wscales.dtype == torch.float32 and torch.equal(model[0].wscales, scales)
    away = copy.deepcopy(model).half().to("meta")
    assert away[0].torch_dtype == torch.float16 and away[0].wscales.dtype == torch.float32
    back = away.to_empty(device="cpu")
    assert back[0].torch_dtype == torch.float16 and back[0].wscales.device.type == "cpu"


def test_codes_of_a_cast_layer_without_a_bias_go_to_its_type(monkeypatch):
    """``forward_quant`` behind ``rms_norm_quantize_w8a8`` names no type: the product is asked for in the layer's."""
    from nunchaku_amd.models import linear

    m = W8A8Linear.from_linear(torch.nn.Linear(96, 40, bias=False, dtype=torch.bfloat16)).half()
    asked = []
    monkeypatch.setattr(linear, "gemm_w8a8", lambda *a, out_dtype=None, **kw: asked.append(out_dtype))
    m.forward_quant(torch.zeros(2, 96, dtype=torch.int8), torch.ones(2))
    assert asked == [torch.float16]
