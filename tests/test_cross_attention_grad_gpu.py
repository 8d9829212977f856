"""Gradients of cross attention against the formulas in 64 bits on the same half inputs, and against
differences of the definition.

Bounds, element by element. dv = sum_i p do: p is off by less than 2^-13 of itself (scores and exponential) and is
rounded to half as 2^12 p (2^-11; below 2^-26 it is subnormal and off by at most 2^-37). dq = scale sum_j ds k
with ds = p (dp - delta): the same 2^-13 of ds, one rounding to half (2^-11, at most 2^-25 where it is subnormal),
p times the error of delta, which is do . (out given - out exact) plus fp32 summation (2^-20 of sum |do out|), and p
times the fp32 summation of dp (2^-20 of sum |do v|). dk likewise with q. Every result is rounded to half once more
(2^-11, at most 2^-25)."""
import math

import pytest
import torch

from niutensor_b200 import capi, ops
from tests.test_cross_attention_gpu import DEV, INF, NAN, lens, make

pytestmark = pytest.mark.gpu


def past(length, n, batch):
    if length is None:
        return torch.zeros(batch, n, dtype=torch.bool, device=DEV)
    return torch.arange(n, device=DEV)[None] >= length.clamp(0, n)[:, None]


def formulas(q, k, v, out, do, ql, kl, scale):
    """[(gradient, bound)] for q, k and v"""
    batch, heads, n, d = q.shape
    kv, m, group = k.shape[1], k.shape[2], heads // k.shape[1]
    pq, pk = past(ql, n, batch)[:, None, :, None], past(kl, m, batch)[:, None, :, None]
    q, do, out = (x.double().masked_fill(pq, 0.0) for x in (q, do, out))
    k, v = (x.double().masked_fill(pk, 0.0).repeat_interleave(group, 1) for x in (k, v))
    s = (q @ k.transpose(2, 3) * scale).masked_fill(pk.transpose(2, 3), -INF)
    lse = torch.logsumexp(s, -1) if m else torch.full(q.shape[:3], -INF, device=DEV, dtype=torch.float64)
    p = torch.exp(s - lse.masked_fill(lse == -INF, 0.0)[..., None]).masked_fill(pq, 0.0)
    o = p @ v
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    e_delta = (do * (out - o)).sum(-1, keepdim=True).abs() + (do * out).abs().sum(-1, keepdim=True) * 2.0 ** -20
    e_ds = ds.abs() * (2.0 ** -11 + 2.0 ** -13) + p * (e_delta + (do.abs() @ v.abs().transpose(2, 3)) * 2.0 ** -20) + 2.0 ** -25
    e_ds = e_ds.masked_fill(pq, 0.0).masked_fill(pk.transpose(2, 3), 0.0)
    e_p = p * (2.0 ** -11 + 2.0 ** -13) + 2.0 ** -37

    def shared(x):
        return x.view(batch, kv, group, m, d).sum(2)
    rows = [(ds @ k * scale, e_ds @ k.abs() * scale), (shared(ds.transpose(2, 3) @ q) * scale, shared(e_ds.transpose(2, 3) @ q.abs()) * scale),
            (shared(p.transpose(2, 3) @ do), shared(e_p.transpose(2, 3) @ do.abs()))]
    return [(x, e + x.abs() * 2.0 ** -11 + 2.0 ** -25) for x, e in rows]


def check(q, k, v, ql=None, kl=None, scale=None, size=0.25, seed=5, split=False):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    do = (torch.randn(q.shape, device=DEV, generator=g) * size).half()
    if split:
        do = do.transpose(1, 2).contiguous().transpose(1, 2)
    if ql is not None:
        do = do.masked_fill(past(ql, q.shape[2], q.shape[0])[:, None, :, None], NAN)
    out, lse = ops.CrossAttention(q, k, v, ql, kl, scale=scale, with_lse=True)
    got = ops.GradCrossAttention(q, k, v, out, lse, do, ql, kl, scale=scale)
    wants = formulas(q, k, v, out, do, ql, kl, 1.0 / math.sqrt(q.shape[3]) if scale is None else scale)
    for name, like, x, (want, bound) in zip("qkv", (q, k, v), got, wants):
        assert x.shape == like.shape and x.dtype == torch.float16 and torch.isfinite(x).all(), name
        worst = ((x.double() - want).abs() / bound).max().item() if x.numel() else 0.0
        assert worst <= 1.0, (name, worst)
    if ql is not None:
        assert (got[0].masked_select(past(ql, q.shape[2], q.shape[0])[:, None, :, None]) == 0).all()
    if kl is not None:
        at = past(kl, k.shape[2], k.shape[0])[:, None, :, None]
        assert (got[1].masked_select(at) == 0).all() and (got[2].masked_select(at) == 0).all()
    assert capi.lib().ntb_device_status(0) == capi.OK
    return out, lse, do, got


@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 1, 8), (2, 2, 2, 1, 130, 64), (2, 2, 1, 130, 1, 128), (1, 2, 2, 64, 64, 64), (1, 2, 2, 128, 128, 128), (2, 4, 2, 127, 129, 128),
    (2, 3, 1, 129, 127, 72), (1, 2, 2, 257, 384, 64), (1, 4, 1, 600, 130, 128), (1, 2, 2, 100, 3000, 128), (1, 1, 1, 3000, 100, 64),
    (1, 1, 1, 1100, 1100, 40), (30, 8, 4, 100, 140, 64), (24, 4, 4, 200, 200, 128),
])
@pytest.mark.parametrize("split", [False, True])
def test_whole_lengths(shape, split):
    check(*make(*shape, split=split), split=split)


@pytest.mark.parametrize("shape,ql,kl", [
    ((6, 2, 2, 150, 300, 64), [150, 0, 1, 128, 129, 7], [300, 10, 0, 128, 127, 1]),
    ((4, 4, 1, 140, 260, 128), [140, 128, 0, 60], [259, 128, 256, 0]),
    ((5, 6, 2, 9, 200, 128), [9, 1, 5, 0, 8], [200, 100, 3, 50, 0]),              # many short tiles, each with rows past the end
    ((2, 8, 1, 100, 1500, 64), [99, 3], [1400, 1]),                               # few key heads, split walks
    ((3, 1, 1, 40, 90, 32), [-4, 99, 40], [90, -1, 1000]),
    ((2, 3, 3, 260, 130, 96), None, [129, 1]),
])
def test_lengths_and_garbage_behind_them(shape, ql, kl):
    for split in (False, True):
        q, k, v = make(*shape, split=split)
        tq, tk = None if ql is None else lens(ql), lens(kl)
        out, lse, do, clean = check(q, k, v, tq, tk, split=split)
        out = out.clone()
        for b, length in enumerate(kl):
            k[b, :, max(0, length):], v[b, :, max(0, length):] = NAN, INF
            if ql is not None:
                for x in (q, do, out):
                    x[b, :, max(0, ql[b]):] = NAN
        again = ops.GradCrossAttention(q, k, v, out, lse, do, tq, tk)
        for a, c in zip(again, clean):
            assert torch.equal(a, c)


def test_empty_sides():
    for n, m in ((5, 0), (0, 5), (0, 0)):
        q, k, v = make(2, 2, 1, n, m, 64)
        out, lse = ops.CrossAttention(q, k, v, with_lse=True)
        for x, like in zip(ops.GradCrossAttention(q, k, v, out, lse, torch.ones_like(q)), (q, k, v)):
            assert x.shape == like.shape and (x == 0).all()


def test_gradients_of_any_size():
    """incoming gradients near half's ends: small ones lose no more than the bound, large ones stay finite"""
    for size in (2.0 ** -14, 2.0 ** -8, 16.0, 300.0):
        check(*make(1, 2, 2, 150, 200, 64), size=size)


def test_against_differences():
    """the directional derivative of sum(out * do), by central differences of the definition in 64 bits"""
    q, k, v = make(1, 2, 1, 70, 90, 64)
    kl = lens([77])
    _, _, do, (dq, dk, dv) = check(q, k, v, None, kl)
    g = torch.Generator(device=DEV)
    g.manual_seed(11)

    def value(q, k, v):
        k, v = k.repeat_interleave(2, 1)[:, :, :77], v.repeat_interleave(2, 1)[:, :, :77]
        return ((torch.softmax(q @ k.transpose(2, 3) / 8.0, -1) @ v) * do.double()).sum().item()
    x = [t.double() for t in (q, k, v)]
    for i, grad in enumerate((dq, dk, dv)):
        u = torch.randn(x[i].shape, device=DEV, dtype=torch.float64, generator=g)
        h = 1e-4
        y = [value(*[t + (sign * h * u if j == i else 0.0) for j, t in enumerate(x)]) for sign in (1, -1)]
        numeric, ours = (y[0] - y[1]) / (2 * h), (grad.double() * u).sum().item()
        # the elements' errors (2^-11 and a little of each, signs at random against u's) add up as their 2-norm does: allow 6 of it
        assert abs(numeric - ours) <= 6 * 2.0 ** -10 * (grad.double() * u).norm().item() + 1e-6 * abs(numeric)


def test_shared_and_broadcast_keys():
    """query heads that share a key head add up; a broadcast k and v gets every copy's gradient"""
    q, k, v = make(2, 6, 2, 80, 100, 64)
    check(q, k, v)
    k1, v1 = k[:1].expand(2, 2, 100, 64), v[:1].expand(2, 2, 100, 64)
    out, lse, do, a = check(q, k1, v1)
    b = ops.GradCrossAttention(q, k1.contiguous(), v1.contiguous(), out, lse, do)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    # dout broadcast over everything, as the gradient of a sum arrives
    one = torch.full((1, 1, 1, 64), 0.5, device=DEV).half()
    x = ops.GradCrossAttention(q, k, v, out, lse, one.expand(2, 6, 1, 64).expand(2, 6, 80, 64).contiguous())
    y = ops.GradCrossAttention(q, k, v, out, lse, one.expand(2, 6, 80, 64).contiguous())
    for s, t in zip(x, y):
        assert torch.equal(s, t)


def test_repeats_streams_and_capture():
    q, k, v = make(3, 4, 2, 140, 500, 128)
    kl, ql = lens([500, 33, 257]), lens([140, 100, 2])
    out, lse, do, first = check(q, k, v, ql, kl)
    do = torch.nan_to_num(do)
    first = [x.clone() for x in ops.GradCrossAttention(q, k, v, out, lse, do, ql, kl)]
    side = torch.cuda.Stream()
    for _ in range(4):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = ops.GradCrossAttention(q, k, v, out, lse, do, ql, kl)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(first, again):
            assert torch.equal(a, b)
    graphs = []
    for _ in range(2):                                # two graphs of the same step, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, l = ops.CrossAttention(q, k, v, ql, kl, with_lse=True)
            res = ops.GradCrossAttention(q, k, v, o, l, do, ql, kl)
        graphs.append((g, res))
    for x in (q, k, v, do):
        x.copy_(torch.randn_like(x))
    graphs[0][0].replay()
    graphs[1][0].replay()
    o, l = ops.CrossAttention(q, k, v, ql, kl, with_lse=True)
    want = ops.GradCrossAttention(q, k, v, o, l, do, ql, kl)
    torch.cuda.synchronize()
    for g, res in graphs:
        for a, b in zip(res, want):
            assert torch.equal(a, b)


def test_a_last_wave_split_over_the_gpu():
    """more items than SMs on either side, the rest of them in a launch of split items"""
    check(*make(10, 16, 16, 100, 1100, 64))
    check(*make(10, 16, 16, 1100, 100, 64), ql=lens([1100, 5, 0, 128, 999, 1, 640, 641, 1100, 77]))


@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 63, 8), (2, 2, 2, 15, 64, 64), (2, 4, 2, 8, 65, 128), (1, 6, 2, 5, 128, 104), (2, 16, 1, 2, 129, 64), (1, 8, 1, 4, 1000, 128),
    (3, 3, 3, 32, 260, 128), (2, 2, 2, 17, 4097, 72), (1, 2, 2, 11, 9000, 40), (60, 8, 8, 15, 243, 104), (1, 4, 4, 32, 1, 128),
])
@pytest.mark.parametrize("split", [False, True])
def test_few_rows(shape, split):
    check(*make(*shape, split=split), split=split)


@pytest.mark.parametrize("shape,ql,kl", [
    ((6, 2, 2, 15, 300, 64), [15, 0, 1, 14, 8, 7], [300, 10, 0, 128, 127, 1]),
    ((5, 6, 2, 9, 200, 128), [9, 1, 5, 0, 8], [200, 100, 3, 50, 0]),
    ((2, 8, 1, 4, 5000, 104), [4, 3], [4400, 1]),                                 # a split walk whose second sentence ends in its first part
    ((3, 1, 1, 32, 90, 32), [-4, 99, 30], [90, -1, 1000]),
    ((2, 4, 4, 3, 700, 128), None, [640, 65]),
])
def test_few_rows_with_lengths_and_garbage_behind_them(shape, ql, kl):
    for split in (False, True):
        q, k, v = make(*shape, split=split)
        tq, tk = None if ql is None else lens(ql), lens(kl)
        out, lse, do, clean = check(q, k, v, tq, tk, split=split)
        out = out.clone()
        for b, length in enumerate(kl):
            k[b, :, max(0, length):], v[b, :, max(0, length):] = NAN, INF
            if ql is not None:
                for x in (q, do, out):
                    x[b, :, max(0, ql[b]):] = NAN
        for a, c in zip(ops.GradCrossAttention(q, k, v, out, lse, do, tq, tk), clean):
            assert torch.equal(a, c)


@pytest.mark.parametrize("rows", [6, 60, 200])
def test_a_row_that_is_infinite(rows):
    """in one sentence it leaves the others, and the keys behind its end, alone"""
    q, k, v = make(3, 2, 2, rows, 100, 64)
    tk = lens([70, 70, 70])
    out, lse, do, clean = check(q, k, v, None, tk)
    do = do.clone()
    do[1, :, 2] = INF
    got = ops.GradCrossAttention(q, k, v, out, lse, do, None, tk)
    for a, c in zip(got, clean):
        assert torch.equal(a[0], c[0]) and torch.equal(a[2], c[2])
    assert (got[1][1, :, 70:] == 0).all() and (got[2][1, :, 70:] == 0).all()


@pytest.mark.parametrize("shape", [
    (60, 4, 4, 100, 50, 128), (60, 4, 4, 130, 120, 64), (2, 4, 4, 32, 100, 128), (1, 3, 3, 64, 128, 104), (2, 2, 2, 33, 65, 72), (1, 1, 1, 50, 64, 40),
    (2, 6, 3, 31, 127, 64), (57, 8, 4, 40, 17, 128), (1, 2, 2, 1, 1, 64), (1, 2, 2, 17, 16, 32), (40, 6, 6, 500, 33, 64), (3, 2, 1, 20, 96, 96),
])
@pytest.mark.parametrize("split", [False, True])
def test_few_keys(shape, split):
    check(*make(*shape, split=split), split=split)


@pytest.mark.parametrize("shape,ql,kl", [
    ((6, 2, 2, 60, 64, 64), [60, 0, 1, 33, 32, 31], [64, 10, 0, 63, 17, 1]),
    ((5, 4, 2, 30, 128, 128), [30, 1, 5, 0, 8], [128, 100, 65, 50, 0]),
    ((80, 3, 3, 150, 60, 104), list(range(71, 151)), list(range(60, -20, -1))),   # no keys or all behind the end, too
    ((3, 1, 1, 32, 90, 32), [-4, 99, 30], [90, -1, 1000]),
    ((2, 4, 4, 64, 120, 64), None, [97, 16]),
])
def test_few_keys_with_lengths_and_garbage_behind_them(shape, ql, kl):
    for split in (False, True):
        q, k, v = make(*shape, split=split)
        tq, tk = None if ql is None else lens(ql), lens(kl)
        out, lse, do, clean = check(q, k, v, tq, tk, split=split)
        out = out.clone()
        for b, length in enumerate(kl):
            k[b, :, max(0, length):], v[b, :, max(0, length):] = NAN, INF
            if ql is not None:
                for x in (q, do, out):
                    x[b, :, max(0, ql[b]):] = NAN
        for a, c in zip(ops.GradCrossAttention(q, k, v, out, lse, do, tq, tk), clean):
            assert torch.equal(a, c)


@pytest.mark.parametrize("n,m,d", [(3, 300, 64), (20, 150, 128), (40, 60, 64), (30, 100, 128), (64, 128, 128), (150, 300, 64)])
def test_every_kernel_takes_broadcasts_far_offsets_and_graphs(n, m, d):
    q, k, v = make(2, 4, 4, n, m, d)
    kl, ql = lens([m, m // 2]), lens([n - 1, n])
    # k and v of one sentence for both, then of one head for all
    for k1, v1 in ((k[:1].expand(2, 4, m, d), v[:1].expand(2, 4, m, d)), (k[:, :1].expand(2, 4, m, d), v[:, :1].expand(2, 4, m, d))):
        out, lse, do, a = check(q, k1, v1, ql, kl)
        for x, y in zip(a, ops.GradCrossAttention(q, k1.contiguous(), v1.contiguous(), out, lse, do, ql, kl)):
            assert torch.equal(x, y)
    # rows, heads and sentences far apart: the last lie behind 2^31 elements
    def far(x):
        rows = x.shape[2]
        pool = torch.empty(2 ** 31 + 2 ** 27, device=DEV, dtype=torch.float16)
        view = pool.as_strided((2, 4, rows, d), (2 ** 31 - 4 * 2 ** 20, 2 ** 20, 2 ** 11, 1), pool.numel() - (2 ** 31 + 3 * 2 ** 20))
        return view.copy_(x)
    do = torch.nan_to_num(do)
    out, lse = ops.CrossAttention(q, k, v, ql, kl, with_lse=True)
    want = ops.GradCrossAttention(q, k, v, out, lse, do, ql, kl)
    for at in range(2):                                   # three of the five, and the other two: each takes 4.5 GB
        qs, ks, vs, os, ds = (far(x) if i % 2 == at else x for i, x in enumerate((q, k, v, out, do)))
        for x, y in zip(ops.GradCrossAttention(qs, ks, vs, os, lse, ds, ql, kl), want):
            assert torch.equal(x, y)
        del qs, ks, vs, os, ds
    # another stream, and two graphs replayed in turn
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.GradCrossAttention(q, k, v, out, lse, do, ql, kl)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = ops.GradCrossAttention(q, k, v, out, lse, do, ql, kl)
        graphs.append((g, res))
    for g, res in graphs:
        g.replay()
    torch.cuda.synchronize()
    for got in (again, graphs[0][1], graphs[1][1]):
        for x, y in zip(got, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("n,m", [(200, 0), (40, 0), (0, 300), (3, 0)])
def test_empty_sides_of_other_sizes(n, m):
    q, k, v = make(2, 4, 2, n, m, 128)
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    for x, like in zip(ops.GradCrossAttention(q, k, v, out, lse, torch.ones_like(q)), (q, k, v)):
        assert x.shape == like.shape and (x == 0).all()
    assert capi.lib().ntb_device_status(0) == capi.OK
