"""GPU: feed-forward blocks whose linears are not both nn.Linear."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("which", [(True, False), (False, True), (True, True)])
def test_either_linear_of_an_ffn(which):
    from datr_amd.fused import ffn_relu
    from datr_amd.int8 import Int8Linear
    torch.manual_seed(3)
    pair = [torch.nn.Linear(256, 512).to(DEV), torch.nn.Linear(512, 256).to(DEV)]
    pair = [Int8Linear(p) if q else p for p, q in zip(pair, which)]
    x = torch.randn(2, 45, 256, device=DEV)
    with torch.no_grad():
        got, want = ffn_relu(x, *pair), pair[1](torch.relu(pair[0](x)))
    assert torch.equal(got, want)


def test_a_linear_of_another_class_takes_the_fused_block():
    from datr_amd.fused import ffn_add_norm

    class Other(torch.nn.Module):
        def __init__(self, linear):
            super().__init__()
            self.weight, self.bias, self.out_features = linear.weight, linear.bias, linear.out_features

        def forward(self, x):
            return torch.nn.functional.linear(x, self.weight, self.bias)

    torch.manual_seed(5)
    pair, norm = [torch.nn.Linear(256, 512).to(DEV), torch.nn.Linear(512, 256).to(DEV)], torch.nn.LayerNorm(256).to(DEV)
    x = torch.randn(90, 256, device=DEV)
    got, want = ffn_add_norm(x, Other(pair[0]), Other(pair[1]), norm), ffn_add_norm(x, *pair, norm)
    assert got is not None and torch.equal(got, want)
