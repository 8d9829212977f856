"""Gradients of cross attention where ds = p (dp - delta) leaves the range of halves though dq and dk do not: many keys
and small incoming gradients, and large ones.

ds goes into the products as halves times a power of two that brings the largest of a row (for dk: of a key's row of a
tile, or of 16 keys' rows) between 2^7 and 2^15. So it is off by 2^-11 of itself, or, where it is less than 2^-21 of that
largest, by at most 2^-25 against 2^7: 2^-32 of it. Besides (as in the other tests of the gradients): scores and
exponential 2^-13, p times the error of delta (of the out that was given, and 2^-20 of sum |do out|) and of dp (2^-20 of
sum |do v|), and the result's own rounding (2^-11, at most 2^-25)."""
import math

import pytest
import torch

from niutensor_b200 import capi, ops
from tests.test_cross_attention_gpu import DEV, INF, make

pytestmark = pytest.mark.gpu

# few rows (whole and split walks), query tiles (whole and split), few keys, shared key heads
SHAPES = [(1, 2, 2, 8, 8192, 64), (1, 8, 2, 5, 4000, 128), (40, 4, 4, 20, 1000, 64), (1, 2, 2, 200, 8192, 64), (8, 8, 2, 150, 4000, 128),
          (1, 1, 1, 64, 16384, 64), (2, 2, 2, 60, 100, 64), (64, 4, 4, 300, 60, 128), (2, 2, 2, 200, 120, 128)]


def formulas(q, k, v, out, do, scale):
    batch, heads, n, d = q.shape
    kv, m, group = k.shape[1], k.shape[2], heads // k.shape[1]
    q, do, out = (x.double() for x in (q, do, out))
    k, v = (x.double().repeat_interleave(group, 1) for x in (k, v))
    p = torch.softmax(q @ k.transpose(2, 3) * scale, -1)
    o = p @ v
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    e_delta = (do * (out - o)).sum(-1, keepdim=True).abs() + (do * out).abs().sum(-1, keepdim=True) * 2.0 ** -20
    e_ds = ds.abs() * (2.0 ** -11 + 2.0 ** -13) + p * (e_delta + (do.abs() @ v.abs().transpose(2, 3)) * 2.0 ** -20)
    row = e_ds + ds.abs().amax(-1, keepdim=True) * 2.0 ** -32                       # of a query: dq
    head = e_ds + ds.abs().view(batch, kv, -1).amax(-1).repeat_interleave(group, 1)[..., None, None] * 2.0 ** -32
    e_p = p * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -37

    def shared(x):
        return x.view(batch, kv, group, m, d).sum(2)
    rows = [(ds @ k * scale, row @ k.abs() * scale), (shared(ds.transpose(2, 3) @ q) * scale, shared(head.transpose(2, 3) @ q.abs()) * scale),
            (shared(p.transpose(2, 3) @ do), shared(e_p.transpose(2, 3) @ do.abs()))]
    return [(x, e + x.abs() * 2.0 ** -11 + 2.0 ** -25) for x, e in rows]


def check(q, k, v, do, scale=None):
    out, lse = ops.CrossAttention(q, k, v, scale=scale, with_lse=True)
    got = ops.GradCrossAttention(q, k, v, out, lse, do, scale=scale)
    for name, x, (want, bound) in zip("qkv", got, formulas(q, k, v, out, do, 1.0 / math.sqrt(q.shape[3]) if scale is None else scale)):
        # what half cannot hold is infinite of the same sign
        fits = want.abs() + bound < 65504.0
        assert torch.isfinite(x[fits]).all(), name
        worst = ((x.double() - want).abs() / bound)[fits].max().item()
        assert worst <= 1.0, (name, worst)
        over = want.abs() - bound > 65520.0
        assert (x[over].double() == want[over].sign() * INF).all(), name
        want16 = want.half().double()
        err, least = ((x.double() - want)[fits]).norm().item(), ((want16 - want)[fits]).norm().item()
        yield name, err, least, want[fits].norm().item()
    assert capi.lib().ntb_device_status(0) == capi.OK


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -10, 2.0 ** -4, 64.0])
def test_incoming_gradients_of_any_size(shape, size):
    q, k, v = make(*shape)
    do = (torch.randn(q.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)) * size).half()
    for name, err, least, norm in check(q, k, v, do):
        # errors of the elements of ds have signs of their own: over all elements at most the result's rounding and a few
        # of ds's (delta's, which is common to a row, included)
        assert err <= 1.5 * least + norm * 2.0 ** -8, (name, err, least, norm)


@pytest.mark.parametrize("shape", SHAPES)
def test_ds_past_the_largest_half(shape):
    """values of some thousands: ds reaches 2^20, dq and dk, with a small scale and small q and k, do not"""
    q, k, v = make(*shape)
    v = v * 1000.0
    do = (torch.randn(q.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(4)) * 200.0).half()
    q, k = q * 2.0 ** -6, k * 2.0 ** -6
    list(check(q, k, v, do, scale=2.0 ** -8))


@pytest.mark.parametrize("shape", SHAPES)
def test_rows_of_very_unequal_gradients(shape):
    """each row of dq keeps its own accuracy beside rows of 2^20 its size; the gradients grow and fall along the walk"""
    q, k, v = make(*shape)
    n = shape[3]
    do = torch.randn(q.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(5))
    for ramp in (torch.linspace(-14.0, 6.0, n, device=DEV), torch.linspace(6.0, -14.0, n, device=DEV)):
        x = (do * torch.exp2(ramp)[None, None, :, None]).half()
        list(check(q, k, v, x))
    # keys whose ds grow from tile to tile, and rows without any gradient first
    x = do.half()
    x[:, :, : n // 2] = 0
    w = (v.float() * torch.linspace(-10.0, 6.0, shape[4], device=DEV).exp2()[None, None, :, None]).half()
    list(check(q, k, w, x))
    list(check(q, k, w.flip(2).contiguous(), x))
    x = torch.zeros_like(x)
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    for g in ops.GradCrossAttention(q, k, v, out, lse, x):
        assert (g == 0).all()


@pytest.mark.parametrize("n,m,d", [(200, 300, 64), (700, 500, 128), (300, 5000, 64)])
def test_ds_that_cancel(n, m, d):
    """ds that are 0 but for roundings: sentences of one key, values that are all alike, incoming gradients across them. What
    little is computed stays as small as the roundings are"""
    from tests.test_cross_attention_gpu import lens
    from tests.test_cross_attention_grad_gpu import check as check_lengths
    q, k, v = make(3, 4, 2, n, m, d)
    check_lengths(q, k, v, None, lens([1, m, 1]))
    check_lengths(q, k, v, lens([n, 130, 5]), lens([1, 2, 129]))
    for size in (1.0, 1000.0):
        same = (v[:, :, :1] * size).expand_as(v).contiguous()
        check_lengths(q, k, same)
        flat = torch.full_like(v, 3.0 * size)                         # do across it: every dp cancels
        do = torch.randn(q.shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6))
        do[..., 1::2] = -do[..., ::2]
        do = do.half()
        out, lse = ops.CrossAttention(q, k, flat, with_lse=True)
        for x in ops.GradCrossAttention(q, k, flat, out, lse, do)[:2]:
            # p times what dp and delta are off by, 2^-20 of sum |do v| each and delta 2^-11 of it for the rounding of out
            limit = (do.double().abs().sum(-1).amax() * 3.0 * size * (2.0 ** -11 + 2.0 ** -19)).item()
            total = n * q.abs().max().item() * 4 if x.shape == k.shape else k.abs().max().item()
            assert torch.isfinite(x).all() and x.abs().max().item() <= limit * total / d ** 0.5 + 2.0 ** -25


@pytest.mark.parametrize("n,m,d", [(4, 300, 64), (40, 60, 64), (200, 300, 64), (300, 5000, 128)])
def test_infinite_ds_reach_the_gradients(n, m, d):
    q, k, v = make(2, 2, 2, n, m, d)
    do = torch.randn_like(q)
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    clean = ops.GradCrossAttention(q, k, v, out, lse, do)
    x = do.clone()
    x[1, 1, n - 1, 3] = INF
    got = ops.GradCrossAttention(q, k, v, out, lse, x)
    assert not torch.isfinite(got[1][1, 1]).any() and not torch.isfinite(got[0][1, 1, n - 1]).any()
    for a, c in zip(got, clean):
        assert torch.equal(a[0], c[0]) and torch.equal(a[1, 0], c[1, 0])
    assert torch.equal(got[0][1, 1, :n - 1], clean[0][1, 1, :n - 1])
