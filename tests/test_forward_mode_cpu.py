"""CPU: operators without a forward-mode derivative refuse an input that carries a tangent; none is dropped in silence."""
import pytest
import torch
from torch.autograd import forward_ad

from datr_amd.distill import topk_distillation_loss
from datr_amd.int8 import linear_int8


def test_the_distillation_loss_refuses_a_tangent():
    z, t, i = torch.zeros(3, 9), torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int64)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            topk_distillation_loss(forward_ad.make_dual(z, torch.ones_like(z)), t, i)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            topk_distillation_loss(forward_ad.make_dual(z, torch.ones_like(z)), t, i)
        with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
            topk_distillation_loss(z, t, i)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda s: topk_distillation_loss(s, t, i), (z,), (z,))


def test_the_8_bit_layer_refuses_a_tangent():
    x, w, s, b = torch.zeros(2, 8), torch.zeros(5, 8, dtype=torch.int8), torch.ones(5), torch.zeros(5)
    with forward_ad.dual_level(), torch.no_grad():
        for n in (0, 2, 3):
            args = [x, w, s, b]
            args[n] = forward_ad.make_dual(args[n], torch.ones_like(args[n]))
            with pytest.raises(RuntimeError, match="no gradient"):
                linear_int8(*args)
        with pytest.raises(RuntimeError, match="Not implemented on the CPU"):
            linear_int8(x, w, s, b)
