"""CPU: a cast of the model (half(), bfloat16(), to(dtype)) leaves an 8-bit layer's scales and bias in 32 bits, where the layer reads them."""
import pytest
import torch

from helpers_int8 import host_layer


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.bfloat16(), lambda m: m.to(torch.float16), lambda m: m.double(),
                                  lambda m: m.half().float(), lambda m: m.to(device="cpu", dtype=torch.bfloat16)])
def test_scales_and_bias_stay_in_32_bits(monkeypatch, cast, bias):
    torch.manual_seed(2)
    layer = host_layer(monkeypatch, 50, 33, bias)
    before = {k: v.clone() for k, v in layer.state_dict().items()}
    model = cast(torch.nn.Sequential(torch.nn.Linear(50, 50), layer))
    after = model[1].state_dict()
    assert before.keys() == after.keys()
    for k, v in before.items():
        assert after[k].dtype == v.dtype and torch.equal(after[k], v)


def test_a_cast_and_a_move_at_once(monkeypatch):
    layer = host_layer(monkeypatch, 50, 33).to("meta", torch.float16)
    assert layer.weight_scale.dtype is torch.float32 and layer.bias.device.type == "meta" and layer.weight.device.type == "meta"


def test_a_checkpoint_saved_in_half_precision(monkeypatch):
    layer = host_layer(monkeypatch, 50, 33)
    state = {k: v if v.dtype is torch.int8 else v.half() for k, v in layer.state_dict().items()}
    for assign in (False, True):
        other = host_layer(monkeypatch, 50, 33)
        other.load_state_dict(state, assign=assign)
        assert other.weight_scale.dtype is torch.float32 and other.bias.dtype is torch.float32
        assert torch.equal(other.weight_scale, state["weight_scale"].float())
