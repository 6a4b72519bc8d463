"""GPU: the distillation loss at the ends of its range of temperatures, against the definition in 64 bits."""
import pytest
import torch

from test_distill_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,k", [(9, 4), (700, 6), (9000, 5), (33000, 20)])
@pytest.mark.parametrize("tau", [1e-30, 1e-25, 1e-21, 1e-6, 1e6, 1e15, 1e18])
def test_small_and_large_temperatures(tau, V, k):
    from datr_amd.distill import topk_distillation_loss
    z, t, index, up = make(6, V, k, torch.float32, V, holes=False)
    z.requires_grad_(True)
    loss = topk_distillation_loss(z, t, index, temperature=tau)
    assert loss.isfinite().all()
    check(z.detach(), t, index, tau, up, loss)
    if tau < 1e-5:
        # the softmaxes are their largest entries, so loss = tau (max z - z of the teacher's first) and the gradient is tau at the one
        # and -tau at the other: the difference, the two products and the sums that add zeros, one rounding each
        first = index.gather(1, t.argmax(1, keepdim=True))
        far = (z.detach().amax(1) - z.detach().gather(1, first)[:, 0]).double()
        assert ((loss.double() - tau * far).abs() <= 8 * 2.0 ** -24 * tau * far).all()
        grad, = torch.autograd.grad(loss, z, up)
        want = torch.zeros_like(z, dtype=torch.float64).scatter_(1, z.argmax(1, keepdim=True), 1.0)
        want.scatter_add_(1, first, -torch.ones_like(first, dtype=torch.float64))
        want *= tau * up.double()[:, None]
        assert ((grad.double() - want).abs() <= 8 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("tau", [1e-30, 1e-3, 1e3, 1e18])
def test_equal_distributions(tau):
    """The student is the teacher and every column is kept: 0 but for the logarithms' and sums' roundings, which tau^2 scales."""
    from datr_amd.distill import topk_distillation_loss
    z, t, index, up = make(6, 12, 12, torch.float32, 5, holes=False)
    loss = topk_distillation_loss(z, z.gather(1, index), index, temperature=tau)
    check(z, z.gather(1, index), index, tau, up, loss)
