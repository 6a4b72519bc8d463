"""CPU: temperatures that the distillation loss refuses, in Python and at its C entry points."""
import pytest
import torch

from datr_amd import _native
from datr_amd.distill import topk_distillation_loss


@pytest.mark.parametrize("tau", [1e-31, 1e19, 1e30, -1e-30])
def test_temperatures_outside_the_range(tau):
    z, t, i = torch.zeros(3, 9), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64)
    with pytest.raises(ValueError, match="temperature"):
        topk_distillation_loss(z, t, i, tau)
    p = 4096                                             # never followed: the calls end at their checks
    assert _native.lib.datr_topk_distill_forward(0, p, 9, 0, p, p, 2, 9, 4, tau, p, p, 0, 0, 0) == -1
    assert _native.lib.datr_topk_distill_backward(0, p, 9, 0, p, p, 2, 9, 4, tau, p, p, p, 0) == -1


@pytest.mark.parametrize("tau", [1e-30, 1e18])
def test_the_ends_are_in_the_range(tau):
    z, t, i = torch.zeros(3, 9), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
        topk_distillation_loss(z, t, i, tau)
    # past the check of tau: there are no rows
    assert _native.lib.datr_topk_distill_forward(0, 0, 9, 0, 0, 0, 0, 9, 4, tau, 0, 0, 0, 0, 0) == 0
