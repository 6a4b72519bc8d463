"""GPU: derivatives of the embedding beyond the first gradient -- forward mode, the gradient's own gradient, forward over reverse,
function transforms -- against nn.Embedding's.  All values are small whole numbers, so every sum is exact in any order."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SIZES = [(40, 10, 16), (3000, 5000, 24), (9000, 700, 8)]


def make(T, V, D, padding_idx=None):
    from datr_amd.embedding import FastEmbedding
    g = torch.Generator().manual_seed(T + V)
    whole = lambda *s: torch.randint(-3, 4, s, generator=g).float().to(DEV)
    own, torchs = FastEmbedding(V, D, padding_idx=padding_idx, scale=2.0).to(DEV), torch.nn.Embedding(V, D, padding_idx=padding_idx).to(DEV)
    with torch.no_grad():
        own.weight.copy_(whole(V, D))
        torchs.weight.copy_(own.weight)
    ids = torch.randint(0, V, (T,), generator=g).to(DEV)
    ids[::5] = 3
    return own, (lambda i: torchs(i) * 2.0), torchs, ids, whole(V, D), whole(T, D)


@pytest.mark.parametrize("padding_idx", [None, 3])
@pytest.mark.parametrize("T,V,D", SIZES)
def test_forward_mode(T, V, D, padding_idx):
    from datr_amd.embedding import embedding, embedding_backward
    own, plain, torchs, ids, along, up = make(T, V, D, padding_idx)
    with forward_ad.dual_level(), torch.no_grad():
        dual = forward_ad.make_dual(own.weight.detach(), along)
        got = forward_ad.unpack_dual(embedding(ids, dual, 2.0, padding_idx))
        assert torch.equal(got.primal, own(ids)) and torch.equal(got.tangent, 2.0 * along[ids])
        # the gradient is linear in its upstream
        grad = forward_ad.unpack_dual(embedding_backward(ids, forward_ad.make_dual(up, 3.0 * up), V, 2.0, padding_idx))
        assert torch.equal(grad.tangent, embedding_backward(ids, 3.0 * up, V, 2.0, padding_idx))
    params = {"weight": own.weight.detach()}
    f = lambda module: lambda p: torch.func.functional_call(module, p, (ids,))
    a, b = torch.func.jvp(f(own), (params,), ({"weight": along},)), torch.func.jvp(f(torchs), (params,), ({"weight": along},))
    assert torch.equal(a[0], 2.0 * b[0]) and torch.equal(a[1], 2.0 * b[1])


@pytest.mark.parametrize("padding_idx", [None, 3])
@pytest.mark.parametrize("T,V,D", SIZES)
def test_the_gradients_gradient(T, V, D, padding_idx):
    """Of sum(up y^2): its gradient, and that one's product with a direction differentiated again."""
    from datr_amd.embedding import embedding
    own, plain, torchs, ids, along, up = make(T, V, D, padding_idx)
    out = []
    for y, weight in ((own, own.weight), (plain, torchs.weight), (lambda i: embedding(i, own.weight, 2.0, padding_idx), own.weight)):
        first, = torch.autograd.grad((up * y(ids).square()).sum(), weight, create_graph=True)
        out.append((first.detach(), torch.autograd.grad((first * along).sum(), weight)[0]))
    for got in (out[0], out[2]):
        assert torch.equal(got[0], out[1][0]) and torch.equal(got[1], out[1][1])
    assert torch.count_nonzero(out[0][1]) > 0
    if padding_idx is not None:
        assert torch.count_nonzero(out[0][0][3]) == 0 and torch.count_nonzero(out[0][1][3]) == 0


@pytest.mark.parametrize("padding_idx", [None, 3])
def test_forward_over_reverse(padding_idx):
    own, plain, torchs, ids, along, up = make(3000, 5000, 24, padding_idx)
    out = []
    for y, weight in ((own, own.weight), (plain, torchs.weight)):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(weight.detach().clone().requires_grad_(True), along)
            module = own if y is own else torchs
            rows = torch.func.functional_call(module, {"weight": dual}, (ids,))
            rows = rows if y is own else 2.0 * rows
            grad, = torch.autograd.grad((up * rows.square()).sum(), dual)
            pair = forward_ad.unpack_dual(grad)
            out.append((pair.primal.detach(), pair.tangent.detach()))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])


def test_function_transforms():
    own, plain, torchs, ids, along, up = make(40, 10, 16, 3)
    several = torch.stack([own.weight.detach(), along, -along])
    f = lambda module: lambda w: torch.func.functional_call(module, {"weight": w}, (ids,))
    assert torch.equal(torch.func.vmap(f(own))(several), 2.0 * torch.func.vmap(f(torchs))(several))
    s = lambda module, by: lambda w: (up * by * f(module)(w)).sum()
    assert torch.equal(torch.func.grad(s(own, 1.0))(along), torch.func.grad(s(torchs, 2.0))(along))
    assert torch.equal(torch.func.vmap(torch.func.grad(s(own, 1.0)))(several), torch.func.vmap(torch.func.grad(s(torchs, 2.0)))(several))
