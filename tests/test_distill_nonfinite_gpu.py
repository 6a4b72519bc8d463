"""GPU: kept logits of the teacher that are not finite, on every path of csrc/distill.hip (16 lanes a row, a wave, a workgroup,
several workgroups).  NaN in a valid slot is an answer that the teacher gave: loss and gradient say so."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V,k", [(9, 1), (9, 4), (700, 1), (700, 4), (5000, 4), (9000, 70), (33000, 20)])
def test_nan_in_valid_slots(V, k, dtype):
    from datr_amd.distill import topk_distillation_loss
    g = torch.Generator().manual_seed(V + k)
    z = torch.randn(7, V, generator=g).to(dtype).to(DEV).requires_grad_(True)
    t = torch.randn(7, k, generator=g).to(dtype).to(DEV)
    index = ((torch.arange(k)[None] * (V // k) + torch.arange(7)[:, None]) % V).to(DEV)
    up = (torch.rand(7, generator=g) + 0.5).to(DEV)
    finite = t.clone()
    nan, inf = float("nan"), float("inf")
    t[0] = nan                                           # nothing but NaN
    t[1] = -inf
    t[1, k // 2] = nan                                   # NaN among -inf
    t[2, k - 1] = nan                                    # NaN beside finite logits
    t[3] = nan
    index[3, 1:] = -1                                    # one valid slot, NaN
    t[4, 0] = inf                                        # no softmax either
    t[5] = -inf                                          # nothing but -inf: the row keeps nothing
    loss = topk_distillation_loss(z, t, index, temperature=2.0)
    grad, = torch.autograd.grad(loss, z, up)
    plain = topk_distillation_loss(z, finite, index, temperature=2.0)
    want, = torch.autograd.grad(plain, z, up)
    assert loss[:5].isnan().all()
    assert loss[5] == 0 and torch.count_nonzero(grad[5]) == 0
    assert loss[6] == plain[6] and torch.equal(grad[6], want[6])
    for r in range(5):
        kept = torch.zeros(V, dtype=torch.bool, device=DEV)
        kept[index[r][index[r] >= 0]] = True
        assert torch.equal(grad[r].isnan(), kept if r != 4 else kept & grad[4].isnan())
        assert grad[r][kept].isnan().any()
        assert torch.equal(grad[r][~kept], want[r][~kept])     # q alone: what the teacher says has no part in it
    with torch.no_grad():
        assert torch.equal(topk_distillation_loss(z, t, index, temperature=2.0).isnan(), loss.isnan())


def test_a_teacher_that_diverged_is_seen():
    """The documented chain: a token of NaN gives a row of NaN logits, of which the top-k selection keeps NaN."""
    from datr_amd.distill import topk_distillation_loss
    from datr_amd.fused import topk_rows
    from datr_amd.int8 import Int8Linear
    torch.manual_seed(1)
    head = Int8Linear(torch.nn.Linear(64, 30).to(DEV))
    x = torch.randn(20, 64, device=DEV)
    x[3, 5] = float("nan")
    with torch.no_grad():
        values, index = topk_rows(head(x), 8)
        loss = topk_distillation_loss(torch.randn(20, 30, device=DEV), values, index)
    assert loss[3].isnan() and int(loss.isnan().sum()) == 1
