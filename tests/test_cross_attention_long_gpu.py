"""Long walks: the tensor core's accumulator rounds toward zero at every instruction, so a sum falls short by an amount
that grows with the walk's length. The walks are split so that it stays below 2^-12 of the sum."""
import pytest
import torch

from niutensor_b200 import capi, ops
from tests.test_cross_attention_gpu import DEV

pytestmark = pytest.mark.gpu


# heads that fill the GPU by themselves (no split is called for by the load), in one and in two query tiles a CTA, and one head
@pytest.mark.parametrize("heads,n,m,d", [(160, 40, 131072, 64), (160, 40, 60000, 128), (160, 256, 131072, 64), (1, 64, 262144, 64), (4, 2, 262144, 64), (320, 2, 1048576, 64)])
def test_sums_of_values_of_one_sign(heads, n, m, d):
    g = torch.Generator(device=DEV).manual_seed(1)
    k = (torch.randn(1, 1, m, d, device=DEV, generator=g) * 0.3).half()
    v = (torch.rand(1, 1, m, d, device=DEV, generator=g) + 0.5).half()
    q = torch.randn(1, heads, n, d, device=DEV, generator=g).half()
    out = ops.CrossAttention(q, k.expand(1, heads, m, d), v.expand(1, heads, m, d))
    total = weight = 0.0
    rows = q[0, ::max(1, heads // 4)].reshape(-1, d).double()
    for i in range(0, m, 1 << 15):
        p = torch.exp(rows @ k[0, 0, i:i + (1 << 15)].double().T / d ** 0.5)
        total, weight = total + p @ v[0, 0, i:i + (1 << 15)].double(), weight + p.sum(1, keepdim=True)
    want = total / weight
    error = out[0, ::max(1, heads // 4)].reshape(-1, d).double() / want - 1.0
    # an element: the sum's shortfall, the weights' roundings (against each other: less than 2^-13 of thousands of them) and the
    # result's (2^-11). The mean: roundings to nearest have signs of their own, 2^-11 over the root of their number, of which
    # six; the shortfall is left
    assert error.abs().max().item() <= 2.0 ** -12 + 2.0 ** -13 + 2.0 ** -11
    assert abs(error.mean().item()) <= 2.0 ** -12 + 6 * 2.0 ** -11 / error.numel() ** 0.5
    assert capi.lib().ntb_device_status(0) == capi.OK


@pytest.mark.parametrize("heads,n,m,d", [(160, 131072, 140, 64), (1, 200000, 300, 64)])
def test_gradients_of_long_queries(heads, n, m, d):
    """dv, a sum over the queries: uniform weights and one incoming gradient, so that it is known"""
    q = torch.zeros(1, 1, n, d, device=DEV).half().expand(1, heads, n, d)
    k = torch.zeros(1, heads, m, d, device=DEV).half()
    v = torch.randn(1, heads, m, d, device=DEV).half()
    do = (torch.rand(1, 1, n, d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)) * 0.1 + 0.05).half()
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    _, _, dv = ops.GradCrossAttention(q, k, v, out, lse, do.expand(1, heads, n, d))
    want = do.double().sum(2, keepdim=True) / m
    error = dv.double() / want - 1.0
    # p = 1 / m rounded to half as 2^12 / m (2^-11, the same in every term), the shortfall and the result's rounding
    p = torch.tensor(4096.0 / m).half().double().item() / 4096.0 * m
    assert (error - (p - 1.0)).abs().max().item() <= 2.0 ** -12 + 2.0 ** -13 + 2.0 ** -11
