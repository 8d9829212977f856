"""A row of the result depends on its own query and its sentence's keys, bit for bit: not on what lies behind the
queries' end, nor on the other rows that a kernel works on beside it."""
import pytest
import torch

from niutensor_b200 import ops
from tests.test_cross_attention_gpu import DEV, INF, NAN, lens

pytestmark = pytest.mark.gpu

# few rows, few rows with split keys, query tiles with split keys, and with whole ones
SHAPES = [(8, 700, 64), (3, 5000, 128), (60, 1500, 64), (200, 900, 128)]


def climbing(n, m, d):
    """scores whose maximum grows slowly, by less than the reference may lag"""
    g = torch.Generator(device=DEV)
    g.manual_seed(9)
    base = torch.randn(1, 1, 1, d, device=DEV, generator=g)
    base = base / base.norm()
    k = (base * torch.linspace(0.0, 8.0, m, device=DEV)[None, None, :, None] + 0.1 * torch.randn(2, 2, m, d, device=DEV, generator=g)).half()
    q = (base * 4.0 + 0.3 * torch.randn(2, 2, n, d, device=DEV, generator=g)).half()
    v = torch.randn(2, 2, m, d, device=DEV, generator=g).half()
    return q, k, v, base


@pytest.mark.parametrize("n,m,d", SHAPES)
@pytest.mark.parametrize("garbage", [3.0, 30.0, 30000.0, INF, NAN])
def test_rows_behind_the_end(n, m, d, garbage):
    q, k, v, base = climbing(n, m, d)
    live = n - n // 3
    ql, kl = lens([live, live - 1]), lens([m, m - 70])
    q[0, :, live:], q[1, :, live - 1:] = 0.0, 0.0
    clean, clean_lse = ops.CrossAttention(q, k, v, ql, kl, scale=0.7, with_lse=True)
    fill = (base * garbage).half() if garbage < 1e4 else torch.full_like(base, garbage).half()
    q[0, :, live:], q[1, :, live - 1:] = fill[0], fill[0]
    out, lse = ops.CrossAttention(q, k, v, ql, kl, scale=0.7, with_lse=True)
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("n,m,d", SHAPES)
def test_other_rows(n, m, d):
    q, k, v, base = climbing(n, m, d)
    clean, clean_lse = ops.CrossAttention(q, k, v, scale=0.7, with_lse=True)
    for size in (3.0, 30.0):
        x = (base * size).half().expand_as(q).clone()
        x[:, :, ::3] = q[:, :, ::3]
        out, lse = ops.CrossAttention(x, k, v, scale=0.7, with_lse=True)
        assert torch.equal(out[:, :, ::3], clean[:, :, ::3]) and torch.equal(lse[:, :, ::3], clean_lse[:, :, ::3])
