"""CPU: what an 8-bit layer loads.  Its integers and their scales belong together; a float checkpoint cast to int8 would be zeros."""
import pytest
import torch

from datr_amd.checkpoint import load_model_state
from helpers_int8 import host_layer


def same(a, b):
    return all(torch.equal(a[k], b[k]) and a[k].dtype == b[k].dtype for k in a) and a.keys() == b.keys()


def test_a_float_checkpoint_is_refused(monkeypatch):
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(50, 50), host_layer(monkeypatch, 50, 33))
    before = {k: v.clone() for k, v in model[1].state_dict().items()}
    floats = torch.nn.Sequential(torch.nn.Linear(50, 50), torch.nn.Linear(50, 33)).state_dict()
    for strict in (True, False):
        with pytest.raises(RuntimeError, match="1.weight.*int8"):
            model.load_state_dict(floats, strict=strict)
    with pytest.raises(RuntimeError, match="1.weight.*int8"):
        load_model_state(model, {"model": floats}, ignore_keywords=["label_enc"])
    assert same(before, model[1].state_dict())
    # what is left out on purpose stays out
    kept = load_model_state(model, {"model": floats}, ignore_keywords=["1."])
    assert sorted(kept.missing_keys) == ["1.bias", "1.weight", "1.weight_scale"] and same(before, model[1].state_dict())


def test_integers_and_scales_are_loaded_together(monkeypatch):
    torch.manual_seed(1)
    a, b = host_layer(monkeypatch, 50, 33), host_layer(monkeypatch, 50, 33)
    before = {k: v.clone() for k, v in a.state_dict().items()}
    for left_out in ("weight", "weight_scale"):
        part = {k: v for k, v in b.state_dict().items() if k != left_out}
        with pytest.raises(RuntimeError, match="belong together"):
            a.load_state_dict(part, strict=False)
        assert same(before, a.state_dict())
    a.load_state_dict(b.state_dict())
    assert same(b.state_dict(), a.state_dict())
    with pytest.raises(RuntimeError, match="size mismatch"):
        host_layer(monkeypatch, 50, 34).load_state_dict(b.state_dict())


@pytest.mark.parametrize("ignore", [[], ["label_enc"]])
def test_a_checkpoint_of_integers_is_no_float_layers(monkeypatch, ignore):
    torch.manual_seed(2)
    model = torch.nn.Sequential(torch.nn.Linear(50, 33))
    before = {k: v.clone() for k, v in model.state_dict().items()}
    integers = torch.nn.Sequential(host_layer(monkeypatch, 50, 33)).state_dict()
    with pytest.raises(RuntimeError, match="0.weight is int8"):
        load_model_state(model, {"model": integers}, ignore_keywords=ignore)
    assert same(before, model.state_dict())
    model[0] = host_layer(monkeypatch, 50, 33)
    load_model_state(model, {"model": integers}, ignore_keywords=ignore)
    assert same(integers, torch.nn.Sequential(model[0]).state_dict())
