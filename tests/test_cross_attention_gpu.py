"""Cross attention against its definition in 64 bits on the same half inputs.

The bound of one output element, with A = sum_j p_j |v_j|: every weight is rounded to half once
(2^-11 of it; below 2^-14 of the running reference it is subnormal and off by at most 2^-25 of the
reference, and the reference is at most the true maximum), the fp32 scores (up to 128 products summed in
fp32, then one multiplication) and the exponential move a weight by less than 2^-13 of itself
for scores of this size, and the result is rounded to half once (2^-11)."""
import math

import pytest
import torch

from niutensor_b200 import capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAN, INF = float("nan"), float("inf")


def make(batch, heads, kv, n, m, d, split=False, seed=1):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def one(h, length):
        shape = (batch, length, h, d) if split else (batch, h, length, d)
        x = torch.randn(shape, device=DEV, generator=g).half()
        return x.transpose(1, 2) if split else x
    return one(heads, n), one(kv, m), one(kv, m)


def lens(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def definition(q, k, v, ql, kl, scale):
    """out, lse and the bound's A and weight of the maximum, all in 64 bits"""
    group, n, m = q.shape[1] // k.shape[1], q.shape[2], k.shape[2]
    q, k, v = (x.double() for x in (q, k, v))
    if kl is not None:
        past = torch.arange(m, device=DEV)[None] >= kl.clamp(0, m)[:, None]
        k = k.masked_fill(past[:, None, :, None], 0.0)
        v = v.masked_fill(past[:, None, :, None], 0.0)
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.nan_to_num(q) @ k.transpose(2, 3) * scale
    if kl is not None:
        s = s.masked_fill(past[:, None, None, :], -INF)
    if m == 0:
        lse = torch.full(q.shape[:3], -INF, device=DEV, dtype=torch.float64)
        top = lse
    else:
        lse, top = torch.logsumexp(s, -1), s.amax(-1)
    safe = lse.masked_fill(lse == -INF, 0.0)
    p = torch.exp(s - safe[..., None])
    out, a, peak = p @ v, p @ v.abs(), torch.exp(top - safe)
    if ql is not None:
        past = torch.arange(n, device=DEV)[None] >= ql.clamp(0, n)[:, None]
        out = out.masked_fill(past[:, None, :, None], 0.0)
        lse = lse.masked_fill(past[:, None, :], -INF)
    return out, lse, a, peak, float(v.abs().max()) if m else 0.0


def check(q, k, v, ql=None, kl=None, scale=None, out=None):
    got, lse = ops.CrossAttention(q, k, v, ql, kl, scale=scale, out=out, with_lse=True)
    alone = ops.CrossAttention(q, k, v, ql, kl, scale=scale)
    assert torch.equal(got, alone)                                       # asking for the statistics changes nothing
    scale = 1.0 / math.sqrt(q.shape[3]) if scale is None else scale
    want, wlse, a, peak, vmax = definition(q, k, v, ql, kl, scale)
    assert got.shape == q.shape and torch.isfinite(got).all()
    bound = a * (2.0 ** -11 + 2.0 ** -13) + want.abs() * 2.0 ** -11 + (k.shape[2] * 2.0 ** -25 * vmax * peak)[..., None] + 2.0 ** -25
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst
    empty = wlse == -INF
    assert torch.equal(lse == -INF, empty)
    assert (got[empty] == 0).all()
    d = (lse.double() - wlse)[~empty]
    assert d.numel() == 0 or (d.abs() <= 2.0 ** -15 + wlse[~empty].abs() * 2.0 ** -20).all()
    assert capi.lib().ntb_device_status(0) == capi.OK
    return got


# (batch, heads, headsKV, lenQ, lenK, d)
@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 1, 8), (1, 8, 8, 1, 23, 64), (2, 4, 4, 1, 64, 64), (2, 4, 4, 1, 65, 128), (3, 5, 1, 3, 127, 72),
    (2, 8, 2, 4, 128, 128), (1, 16, 1, 2, 129, 64), (2, 6, 2, 10, 1000, 40), (1, 2, 1, 16, 4097, 128),         # step kernel
    (1, 1, 1, 33, 1, 8), (2, 2, 2, 61, 73, 64), (1, 3, 1, 127, 128, 128), (2, 4, 2, 128, 129, 64), (1, 2, 2, 129, 255, 128),
    (2, 2, 1, 257, 384, 96), (1, 2, 2, 40, 3000, 128), (1, 1, 1, 300, 2049, 64), (30, 8, 4, 300, 200, 64), (25, 6, 6, 260, 140, 120),
])
@pytest.mark.parametrize("split", [False, True])
def test_whole_lengths(shape, split):
    check(*make(*shape, split=split))


@pytest.mark.parametrize("shape,ql,kl", [
    ((6, 4, 2, 5, 200, 64), None, [0, 1, 63, 64, 65, 200]),
    ((5, 2, 2, 1, 700, 128), [1, 0, 1, 1, 1], [700, 300, 0, 17, 129]),
    ((6, 2, 2, 150, 300, 64), [150, 0, 1, 128, 129, 7], [300, 10, 0, 128, 127, 1]),
    ((4, 4, 1, 140, 260, 128), [140, 128, 0, 60], [259, 128, 256, 0]),
    ((40, 8, 8, 200, 200, 128), [200 - 5 * i for i in range(40)], [5 * i + 1 for i in range(40)]),
    ((3, 2, 2, 50, 5000, 128), [50, 20, 50], [5000, 4097, 3]),
    ((3, 1, 1, 40, 90, 32), [-4, 99, 40], [90, -1, 1000]),                     # clamped to the extents
])
def test_lengths_and_garbage_behind_them(shape, ql, kl):
    """what lies behind a sequence's end -- NaN, infinities -- reaches nothing"""
    for split in (False, True):
        q, k, v = make(*shape, split=split)
        clean = check(q, k, v, None if ql is None else lens(ql), lens(kl))
        for b, length in enumerate(kl):
            length = max(0, length)
            k[b, :, length:], v[b, :, length:] = NAN, INF
            v[b, :, length::2] = NAN
            if ql is not None:
                q[b, :, max(0, ql[b]):] = NAN
        again = ops.CrossAttention(q, k, v, None if ql is None else lens(ql), lens(kl))
        assert torch.equal(clean, again)


def test_no_keys_no_queries_no_batch():
    q, k, v = make(2, 2, 2, 5, 0, 64)
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    assert (out == 0).all() and (lse == -INF).all()
    q, k, v = make(2, 2, 1, 70, 0, 64)
    out, lse = ops.CrossAttention(q, k, v, with_lse=True)
    assert (out == 0).all() and (lse == -INF).all()
    for shape in ((2, 2, 2, 0, 5, 64), (0, 2, 2, 3, 5, 64)):
        q, k, v = make(*shape)
        assert ops.CrossAttention(q, k, v).shape == q.shape


@pytest.mark.parametrize("n", [2, 100, 300])
def test_sharp_and_flat_scores(n):
    """the maximum far ahead, growing from tile to tile, and all keys alike"""
    q, k, v = make(1, 2, 2, n, 900, 64)
    ramp = torch.linspace(0.01, 6.0, 900, device=DEV)[None, None, :, None]
    base = torch.randn(1, 1, 1, 64, device=DEV)
    k = (base * ramp).half().expand(1, 2, 900, 64).contiguous()
    q = base.half().expand(1, 2, n, 64).contiguous()
    check(q, k, v)
    check(q, k.flip(2).contiguous(), v)
    check(-q, k, v)
    check(q, torch.zeros_like(k), v)


def test_scores_of_large_magnitude_stay_finite():
    q, k, v = make(1, 2, 2, 200, 300, 64)
    q, k = q * 200.0, k * 100.0
    out = ops.CrossAttention(q, k, v)
    # differences between scores are in the hundreds: every row is its best key's value, unless two tie nearly
    s = q.double() @ k.double().transpose(2, 3) / 8.0
    top2 = s.topk(2, dim=-1)
    clear = top2.values[..., 0] - top2.values[..., 1] > 40.0
    want = torch.gather(v, 2, top2.indices[..., :1].expand(-1, -1, -1, 64))
    assert clear.any() and torch.isfinite(out).all()
    # The reference of a row is its maximum rounded to fp32 (here up to 2^21, so off by up to 2^-3 in the
    # exponent): the best key's weight w = 2^x, |x| <= 1/8, need not be 1. w is rounded to half for the second
    # product and not for the sum, so out = v * half(w) / w, off by at most 2^-11, and then rounded to half once more.
    a, b = out[clear].double(), want[clear].double()
    assert ((a - b).abs() <= b.abs() * (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -21)).all()


def test_strides_offsets_and_broadcast():
    q, k, v = make(3, 4, 2, 70, 90, 64)
    want = ops.CrossAttention(q, k, v)
    # columns of a wider buffer, at an offset of eight elements; every second row
    wide = torch.randn(3, 4, 140, 160, device=DEV).half()
    view = wide[:, :, ::2, 8:72]
    view.copy_(q)
    assert torch.equal(ops.CrossAttention(view, k, v), want)
    # k and v side by side in one projection
    both = torch.randn(3, 90, 2, 2, 64, device=DEV).half()
    kk, vv = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    kk.copy_(k)
    vv.copy_(v)
    assert torch.equal(ops.CrossAttention(q, kk, vv), want)
    # an output of the caller's, by position instead of by head; the bytes around it stay
    buf = torch.full((3, 72, 4, 64), 7.0, device=DEV).half()
    out = buf[:, 1:71].transpose(1, 2)
    got = ops.CrossAttention(q, k, v, out=out)
    assert got is out and torch.equal(out, want) and (buf[:, 0] == 7).all() and (buf[:, 71] == 7).all()
    # one sentence's states for every row of the batch, one key head for all: strides of 0
    k1, v1 = k[:1].expand(3, 2, 90, 64), v[:1].expand(3, 2, 90, 64)
    assert torch.equal(ops.CrossAttention(q, k1, v1), ops.CrossAttention(q, k1.contiguous(), v1.contiguous()))
    k2, v2 = k[:, :1].expand(3, 2, 90, 64), v[:, :1].expand(3, 2, 90, 64)
    q4 = q[:, :, :3]
    assert torch.equal(ops.CrossAttention(q4, k2, v2), ops.CrossAttention(q4.contiguous(), k2.contiguous(), v2.contiguous()))
    q5 = q[:1].expand(3, 4, 70, 64)
    assert torch.equal(ops.CrossAttention(q5, k, v), ops.CrossAttention(q5.contiguous(), k, v))


def test_last_row_and_column_extents_end_inside_a_tile():
    """head sizes that fill a box only in part: columns behind them are not written"""
    for d in (8, 24, 72, 120):
        for n in (3, 130):
            q, k, v = make(2, 2, 2, n, 150, d)
            buf = torch.full((2, 2, n, 128), 5.0, device=DEV).half()
            check(q, k, v, out=buf[..., :d])
            assert (buf[..., d:] == 5).all()


def test_long_caches_pass_32_bit_offsets():
    """the last sentence's states start beyond 2^31 elements"""
    batch, kv, m, d = 3, 1, 5_700_000, 128
    k = torch.zeros(batch, kv, m, d, device=DEV, dtype=torch.float16)
    v = torch.zeros(batch, kv, m, d, device=DEV, dtype=torch.float16)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    keys = 300
    k[2, 0, m - keys:] = torch.randn(keys, d, device=DEV, generator=g).half()
    v[2, 0, m - keys:] = torch.randn(keys, d, device=DEV, generator=g).half()
    # a window of the cache, as its own view, against the same values moved to a small buffer
    kw, vw = k[:, :, m - keys:], v[:, :, m - keys:]
    for n in (2, 64):
        q = torch.randn(batch, 2, n, d, device=DEV, generator=g).half()
        assert torch.equal(ops.CrossAttention(q, kw, vw), ops.CrossAttention(q, kw.contiguous(), vw.contiguous()))


def test_other_streams_capture_and_repeats():
    q, k, v = make(4, 8, 8, 100, 120, 64)
    q1 = q[:, :, :1].contiguous()
    want, want1 = ops.CrossAttention(q, k, v), ops.CrossAttention(q1, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a, a1 = ops.CrossAttention(q, k, v), ops.CrossAttention(q1, k, v)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, want) and torch.equal(a1, want1)
    out, out1 = torch.empty_like(q), torch.empty_like(q1)
    kl = lens([120, 60, 1, 77])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.CrossAttention(q, k, v, None, kl, out=out)
        ops.CrossAttention(q1, k, v, None, kl, out=out1)
    q.copy_(torch.randn_like(q))
    q1.copy_(q[:, :, :1])
    kl.copy_(lens([3, 120, 119, 0]))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.CrossAttention(q, k, v, None, kl))
    assert torch.equal(out1, ops.CrossAttention(q1, k, v, None, kl))
    first = ops.CrossAttention(q, k, v)
    for _ in range(5):
        assert torch.equal(ops.CrossAttention(q, k, v), first)


def test_agrees_with_the_fused_self_attention():
    """the existing fused attention computes the same where both apply"""
    q, k, v = make(2, 4, 4, 200, 256, 64)
    a, b = ops.CrossAttention(q, k, v), ops.ScaledDotProductAttention(q, k, v)
    assert (a.double() - b.double()).norm() / b.double().norm() <= 2e-3


def test_a_last_wave_split_over_the_gpu():
    """more long items than SMs, the rest of them in a launch of split items"""
    check(*make(5, 16, 16, 150, 3000, 64))
    check(*make(10, 16, 16, 200, 2950, 64), kl=lens([2950, 100, 1, 2000, 0, 2950, 129, 64, 2900, 17]))


def test_two_devices_are_told_apart():
    """the tensors' device counts, not the current one"""
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    q, k, v = (x.to("cuda:1") for x in make(1, 2, 2, 3, 40, 64))
    assert ops.CrossAttention(q, k, v).device == q.device
