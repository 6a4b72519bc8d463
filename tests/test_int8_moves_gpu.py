"""GPU: an 8-bit layer that was moved, called first inside a graph's capture and from two streams at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def moved_layer(seed):
    from datr_amd.int8 import Int8Linear
    torch.manual_seed(seed)
    layer = Int8Linear(torch.nn.Linear(50, 33).to(DEV))
    x = torch.randn(7, 50, device=DEV)
    return layer, x, layer(x).clone()


def test_the_first_call_of_a_moved_layer_is_captured():
    warm, x, want = moved_layer(5)
    layer, _, _ = moved_layer(5)
    layer = layer.cpu().to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        warm(x)                                          # the kernels are loaded, this layer has not been called
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    held = layer.weight
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
    assert layer.weight is held
    assert torch.equal(layer(x), want)                   # before any replay
    for n in range(3):
        x2 = torch.randn(7, 50, device=DEV)
        x.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, warm(x2)) and torch.equal(layer(x2), warm(x2))


def test_the_first_calls_of_a_moved_layer_on_two_streams():
    layer, x, want = moved_layer(6)
    layer = layer.cpu().to(DEV)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(layer(x))
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


def test_loading_after_an_inference_pass():
    layer, x, want = moved_layer(7)
    state = {k: v.clone() for k, v in layer.state_dict().items()}
    layer = layer.cpu().to(DEV)
    with torch.inference_mode():
        assert torch.equal(layer(x), want)
    layer.load_state_dict(state)
    assert torch.equal(layer(x), want)
