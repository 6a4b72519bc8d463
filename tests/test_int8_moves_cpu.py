"""CPU: an 8-bit layer's rows stay at 16-byte borders wherever the layer goes, and a forward pass changes nothing of the layer -- a
buffer bound anew inside a captured call would be memory that only a replay writes."""
import copy

import pytest
import torch

from datr_amd.int8 import Int8Linear
from helpers_int8 import host_layer


def test_a_move_lays_the_rows_out_again(monkeypatch):
    layer = host_layer(monkeypatch, 50, 33)
    before = layer.weight.clone()
    assert copy.deepcopy(layer).weight.stride(0) % 16 == 0
    moved = torch.nn.Sequential(layer).to("meta")[0]
    assert moved.weight.shape == (33, 50) and moved.weight.stride() == (64, 1) and moved.weight.dtype is torch.int8
    layer = host_layer(monkeypatch, 50, 33)
    before = layer.weight.clone()
    layer._apply(lambda t: t.clone())                    # packs the rows, as every copy to another device does
    assert torch.equal(layer.weight, before) and layer.weight.stride(0) % 16 == 0
    even = host_layer(monkeypatch, 64, 33)
    even._apply(lambda t: t.clone())
    assert even.weight.stride() == (64, 1)


def test_assigned_rows_are_laid_out(monkeypatch):
    a, b = host_layer(monkeypatch, 50, 33), host_layer(monkeypatch, 50, 33)
    packed = {k: v.clone() for k, v in b.state_dict().items()}
    assert packed["weight"].stride(0) == 50
    a.load_state_dict(packed, assign=True)
    assert torch.equal(a.weight, b.weight) and a.weight.stride(0) % 16 == 0


def test_a_forward_pass_changes_nothing(monkeypatch):
    layer = host_layer(monkeypatch, 50, 33)
    layer.weight = packed = layer.weight.clone()         # rows 50 bytes apart
    held = {k: (v, v._version) for k, v in layer.named_buffers()}
    with torch.no_grad(), pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        layer(torch.zeros(2, 50))
    assert layer.weight is packed
    for k, v in layer.named_buffers():
        assert v is held[k][0] and v._version == held[k][1]
    assert isinstance(layer, Int8Linear)
