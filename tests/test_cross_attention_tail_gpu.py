"""A dominating key over a long tail of light ones.

The weights of the second product are halves with the running reference taken off. The reference is at most 2^-7 of the
largest weight, so a weight of 2^-21 of it is a normal half (off by 2^-11 of itself), and a lighter one off by at most
2^-25 of the reference, 2^-32 of the largest."""
import math

import pytest
import torch

from niutensor_b200 import ops
from tests.test_cross_attention_gpu import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,m,d", [(1, 32768, 64), (4, 131072, 64), (40, 32768, 64), (150, 40000, 128)])
@pytest.mark.parametrize("nats", [10.0, 16.0, 17.4])
@pytest.mark.parametrize("first", [True, False])
def test_the_tail_keeps_its_mass(n, m, d, nats, first):
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    q = torch.zeros(1, 1, n, d, device=DEV).half()
    q[..., 0] = 1.0
    k = torch.zeros(1, 1, m, d, device=DEV).half()
    at = 3 if first else m - 2
    k[0, 0, at, 0] = nats
    v = (torch.rand(1, 1, m, d, device=DEV, generator=g) + 15.0).half()
    v[0, 0, at] = 0.25
    out, lse = ops.CrossAttention(q, k, v, scale=1.0, with_lse=True)
    s = (q.double() @ k.double().transpose(2, 3))
    p = torch.softmax(s, -1)
    want = p @ v.double()
    # the weights' and scores' roundings, the result's, and the tail's
    bound = want * (2.0 ** -11 + 2.0 ** -13) + want * 2.0 ** -11 + m * 2.0 ** -32 * 16.0 * p.amax(-1, keepdim=True)
    worst = ((out.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst
    assert ((lse.double() - torch.logsumexp(s, -1)).abs() <= 2.0 ** -15).all()


@pytest.mark.parametrize("n", [2, 100, 300])
def test_weights_stay_below_the_largest_half(n):
    """scores that climb by less than the reference's lag at a time: the weights it lets stand, and their sums, are finite"""
    m, d = 4096, 64
    for climb in (0.5, 5.0, 10.3, 11.0):
        q = torch.zeros(1, 2, n, d, device=DEV).half()
        q[..., 0] = 1.0
        k = torch.zeros(1, 2, m, d, device=DEV).half()
        k[..., 0] = (torch.arange(m, device=DEV) // 64).float().mul(climb).half()
        v = torch.ones(1, 2, m, d, device=DEV).half() * 3.0
        out, lse = ops.CrossAttention(q, k, v, scale=1.0, with_lse=True)
        s = q.double() @ k.double().transpose(2, 3)
        want = torch.logsumexp(s, -1)
        # every value is 3: roundings of the weights against their sum, and the result's
        assert ((out.double() - 3.0).abs() <= 3.0 * (2.0 ** -11 + 2.0 ** -13 + 2.0 ** -11) + 3.0 * m * 2.0 ** -32).all()
        assert ((lse.double() - want).abs() <= 2.0 ** -15 + want.abs() * 2.0 ** -20).all()
