"""Calls without query heads: nothing reads k and v, so their gradients are zeros, written as always."""
import pytest
import torch

from niutensor_b200 import capi, ops
from tests.test_cross_attention_gpu import DEV, NAN, lens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m,d", [(5, 7, 64), (1, 300, 128), (200, 40, 64), (40, 300, 8)])
def test_gradients_without_query_heads(n, m, d):
    q = torch.empty(2, 0, n, d, device=DEV).half()
    k, v = (torch.randn(2, 3, m, d, device=DEV).half() for _ in range(2))
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    assert out.shape == q.shape and lse.shape == q.shape[:3]
    for kl in (None, lens([m, m // 2])):
        keep = [torch.full((2, 3, m, d), NAN, device=DEV).half() for _ in range(2)]     # what the allocator hands out next
        del keep
        dq, dk, dv = ops.GradCrossAttention(q, k, v, out, lse, torch.empty_like(q), None, kl)
        assert dq.shape == q.shape and (dk == 0).all() and (dv == 0).all()
    assert capi.lib().ntb_device_status(0) == capi.OK
