"""GPU: scales of which the product leaves the 32-bit range while the result does not."""
import pytest
import torch

from test_int8_gpu import check

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
# a token, few tokens, every tile shape
SIZES = [(1, 256, 40), (12, 256, 40), (40, 256, 40), (40, 256, 8200), (150, 256, 70), (600, 256, 1030), (1100, 256, 4096), (4111, 256, 4001)]


@pytest.mark.parametrize("M,K,N", SIZES)
def test_products_of_scales_out_of_range(M, K, N):
    from datr_amd.int8 import linear_int8
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    ws, bias = torch.rand(N, generator=g) * 0.01 + 1e-3, torch.randn(N, generator=g)
    w[1] = 0                                             # sums of 0 ...
    ws[1] = 1e20                                         # ... under a scale whose product with a large token's is infinite
    w[2] = 127
    ws[2], bias[2] = 1e-17, 0.0                          # with a small token's: subnormal
    ws[3] = 0.0
    bias[5] = 0.0
    x[0] = 1e-23
    if M > 2:
        x[1] *= 1e30
        x[2] = 0
    x, w, ws, bias = (t.to(DEV) for t in (x, w, ws, bias))
    y = linear_int8(x, w, ws, bias)
    check(y, x, w, ws, bias, False)
    assert torch.equal(y[:, 1], bias[1].expand(M)) and torch.equal(y[:, 3], bias[3].expand(M))
    for r in {0, min(1, M - 1), min(2, M - 1), M - 1}:   # and a token alone gives the same
        assert torch.equal(linear_int8(x[r:r + 1], w, ws, bias)[0], y[r])
    # ordinary scales beside them are the same as without them
    some = torch.arange(4, N, device=DEV)
    rows = torch.arange(3 if M > 2 else 0, M, device=DEV)
    if M > 3:
        assert torch.equal(linear_int8(x[rows], w[some], ws[some], bias[some]), y[rows][:, some])


@pytest.mark.parametrize("M,K,N", [s for s in SIZES if s[0] > 2])
def test_the_largest_and_the_smallest_tokens_side_by_side(M, K, N):
    """Tokens of the type's largest magnitude, of 1e30 (on either side of where the kernels share the factors out otherwise) and of
    1e-30, over channels of 1e-6, 1e38 and infinity."""
    from datr_amd.int8 import linear_int8
    g = torch.Generator().manual_seed(M + 1)
    x = torch.randn(M, K, generator=g)
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    ws, bias = torch.rand(N, generator=g) * 1e-6 + 1e-7, torch.randn(N, generator=g)
    x[0] = torch.finfo(torch.float32).max
    x[1] = 2.0 ** 103                                    # scales above and below 2^96
    x[2] = 2.0 ** 102
    x[3:6] *= 1e-30
    w[1], ws[1] = 0, 1e38                                # 0, whatever the scales
    w[2], ws[2] = 127, 1e-30
    w[3], ws[3] = 0, float("inf")                        # the formula's NaN
    x, w, ws, bias = (t.to(DEV) for t in (x, w, ws, bias))
    y = linear_int8(x, w, ws, bias)
    assert torch.equal(y[:, 1], bias[1].expand(M)) and y[:, 3].isnan().all()
    some = torch.tensor([n for n in range(N) if n != 3], device=DEV)
    check(y[:, some], x, w[some], ws[some], bias[some], False)
    for r in (0, 1, 2, 3, M - 1):
        alone = linear_int8(x[r:r + 1], w, ws, bias)[0]
        assert torch.equal(alone[some], y[r][some])
