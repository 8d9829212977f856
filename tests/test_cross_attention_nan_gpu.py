"""What is not finite in a live row or key reaches the result: zeros and a lse of minus infinity stand for rows
without keys, and for nothing else, whichever kernel takes the call."""
import pytest
import torch

from niutensor_b200 import capi, ops
from tests.test_cross_attention_gpu import DEV, INF, NAN, lens, make

pytestmark = pytest.mark.gpu

# the step's kernel with whole and with split keys, query tiles with split and with whole keys, one and two to a CTA
SHAPES = [(1, 2, 2, 3, 40, 64), (1, 2, 1, 2, 3000, 128), (2, 4, 2, 9, 700, 64), (1, 2, 2, 200, 90, 64), (1, 1, 1, 130, 2500, 128), (40, 8, 8, 300, 200, 64)]


def others(x, row):
    return torch.cat((x[:, :, :row], x[:, :, row + 1:]), 2)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bad", [NAN, INF])
def test_a_query_row(shape, bad):
    """its scores are NaN, or infinities of both signs: the formula gives NaN, and every other row what it was"""
    q, k, v = make(*shape)
    clean, clean_lse = ops.CrossAttention(q, k, v, with_lse=True)
    for row in (0, shape[3] - 1):
        x = q.clone()
        x[-1, -1, row] = bad
        out, lse = ops.CrossAttention(x, k, v, with_lse=True)
        assert out[-1, -1, row].isnan().all() and lse[-1, -1, row].isnan()
        out[-1, -1, row], lse[-1, -1, row] = clean[-1, -1, row], clean_lse[-1, -1, row]
        assert torch.equal(others(out, row), others(clean, row)) and torch.equal(others(lse, row), others(clean_lse, row))
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
    assert capi.lib().ntb_device_status(0) == capi.OK


@pytest.mark.parametrize("shape", SHAPES)
def test_a_key_and_a_value(shape):
    """one key of NaN makes every row of its head NaN; one value of NaN its column of the result, not the statistics"""
    q, k, v = make(*shape)
    clean, clean_lse = ops.CrossAttention(q, k, v, with_lse=True)
    heads = shape[1] // shape[2]
    for at in (0, shape[4] // 2, shape[4] - 1):
        x = k.clone()
        x[-1, -1, at] = NAN
        out, lse = ops.CrossAttention(q, x, v, with_lse=True)
        assert out[-1, -heads:].isnan().all() and lse[-1, -heads:].isnan().all()
        assert torch.equal(out[:-1], clean[:-1]) and torch.equal(out[-1, :-heads], clean[-1, :-heads])
        x = v.clone()
        x[-1, -1, at, 5] = NAN
        out, lse = ops.CrossAttention(q, k, x, with_lse=True)
        assert out[-1, -heads:, :, 5].isnan().all() and torch.equal(lse, clean_lse)
        out[-1, -heads:, :, 5] = clean[-1, -heads:, :, 5]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("shape", SHAPES)
def test_keys_of_nan_in_one_part(shape):
    """all keys of a half of the walk: whole warps, tiles and parts of a split walk see nothing else"""
    q, k, v = make(*shape)
    m = shape[4]
    for lo, hi in ((0, m // 2), (m // 2, m), (0, m)):
        x = k.clone()
        x[:, :, lo:hi] = NAN
        out, lse = ops.CrossAttention(q, x, v, with_lse=True)
        assert out.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("shape", SHAPES)
def test_scores_of_minus_infinity(shape):
    """some keys: their weights are 0, as if they were not there. All keys: the quotient 0 / 0"""
    q, k, v = make(*shape)
    q[..., 0] = 1.0
    m = shape[4]
    for lo, hi in ((0, m // 2), (m // 2, m)):
        x = k.clone()
        x[:, :, lo:hi, 0] = -INF
        out, lse = ops.CrossAttention(q, x, v, with_lse=True)
        keep = torch.cat((torch.arange(0, lo), torch.arange(hi, m))).to(DEV)
        s = q.double() @ k.repeat_interleave(shape[1] // shape[2], 1)[:, :, keep].double().transpose(2, 3) / shape[5] ** 0.5
        p = torch.softmax(s, -1)
        w = v.repeat_interleave(shape[1] // shape[2], 1)[:, :, keep].double()
        want = p @ w
        # a weight's rounding and its score's (2^-11, 2^-13), the result's rounding; weights below 2^-14 of a reference that
        # is at most the largest score: 2^-25 each
        bound = (p @ w.abs()) * (2.0 ** -11 + 2.0 ** -13) + want.abs() * 2.0 ** -11 + m * 2.0 ** -25 * w.abs().max() * p.amax(-1, keepdim=True) + 2.0 ** -25
        assert ((out.double() - want).abs() <= bound).all()
        assert ((lse.double() - torch.logsumexp(s, -1)).abs() <= 2.0 ** -15).all()
    k[..., 0] = -INF
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    assert out.isnan().all() and (lse == -INF).all()


def test_lengths_still_decide_what_is_empty():
    """NaN behind the ends, rows without keys and rows behind the end: zeros and minus infinity"""
    for shape in ((3, 4, 2, 4, 900, 64), (3, 2, 2, 150, 900, 64)):
        q, k, v = make(*shape)
        n, m = shape[3], shape[4]
        ql, kl = lens([n, n - 1, n]), lens([m, m - 100, 0])
        clean, clean_lse = ops.CrossAttention(q, k, v, ql, kl, with_lse=True)
        q[1, :, n - 1:], q[2] = NAN, NAN
        k[1, :, m - 100:], v[1, :, m - 100:], k[2], v[2] = NAN, NAN, NAN, NAN
        out, lse = ops.CrossAttention(q, k, v, ql, kl, with_lse=True)
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)
        assert (out[2] == 0).all() and (lse[2] == -INF).all() and (out[1, :, n - 1:] == 0).all() and (lse[1, :, n - 1:] == -INF).all()


@pytest.mark.parametrize("n,m,d", [(3, 300, 64), (3, 3000, 128), (40, 60, 64), (150, 300, 64), (150, 2500, 128)])
def test_gradients_of_a_row_that_is_nan(n, m, d):
    """its dq, and dk and dv of its head; the rest is what it was"""
    q, k, v = make(2, 2, 2, n, m, d)
    do = torch.randn_like(q)

    def step(q):
        out, lse = ops.CrossAttention(q, k, v, with_lse=True)
        return ops.GradCrossAttention(q, k, v, out, lse, do)
    clean = step(q)
    x = q.clone()
    x[1, 1, n - 1] = NAN
    got = step(x)
    assert got[0][1, 1, n - 1].isnan().all() and got[1][1, 1].isnan().all() and got[2][1, 1].isnan().all()
    assert torch.equal(got[0][1, 1, :n - 1], clean[0][1, 1, :n - 1])
    for a, c in zip(got, clean):
        assert torch.equal(a[0], c[0]) and torch.equal(a[1, 0], c[1, 0])
