"""Embedding rows and their gradient against 64-bit sums of the same inputs.

Forward: one fused multiply-add in fp32 (2^-24 of the result) and one rounding to the result's type
(2^-11 for halves, at most 2^-25; none for floats). Gradient: a word's n rows are added one after the other in
fp32, so its sum is off by at most n 2^-24 of the sum of magnitudes, then one multiply-add and one
rounding."""
import pytest
import torch

from niutensor_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, F32 = torch.float16, torch.float32


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def rounding(x, t):
    return x.abs() * 2.0 ** -11 + 2.0 ** -25 if t == F16 else x.abs() * 2.0 ** -24


@pytest.mark.parametrize("t", [F16, F32])
@pytest.mark.parametrize("shape,vocab,d", [((1,), 1, 1), ((3, 7), 11, 8), ((64,), 500, 512), ((5, 13), 900, 513), ((2, 3, 10), 70, 300),
                                           ((4096,), 32000, 1024), ((33,), 50, 2050)])
def test_rows(t, shape, vocab, d):
    g = gen(1)
    w = torch.randn(vocab, d, device=DEV, generator=g).to(t)
    ids = torch.randint(0, vocab, shape, device=DEV, generator=g, dtype=torch.int32)
    pos = torch.randn(shape[-1], d, device=DEV, generator=g).to(t)
    for scale, p in ((1.0, None), (22.627417, pos), (-0.5, pos)):
        got = ops.Embedding(w, ids, scale, p)
        want = w.double()[ids.long()] * torch.tensor(scale, dtype=F32).double().item() + (0.0 if p is None else p.double())
        assert got.shape == want.shape and got.dtype == t
        assert ((got.double() - want).abs() <= rounding(want, t) + want.abs() * 2.0 ** -24).all()
    assert torch.equal(ops.Embedding(w, ids), w[ids.long()])


def test_ids_outside_are_padding_and_rows_may_be_pitched():
    g = gen(2)
    for t, d in ((F16, 64), (F32, 36), (F16, 33)):
        wide = torch.randn(40, 100, device=DEV, generator=g).to(t)
        w = wide[:, 8:8 + d]
        pos = torch.randn(6, d, device=DEV, generator=g).to(t)
        ids = torch.tensor([[0, 39, 40, -1, 2 ** 31 - 1, -2 ** 31], [5, 5, 5, 1, 38, 7]], dtype=torch.int32, device=DEV)
        got = ops.Embedding(w, ids, 2.0, pos)
        ok = (ids >= 0) & (ids < 40)
        want = (w.double()[ids.clamp(0, 39).long()] * 2.0).masked_fill(~ok[..., None], 0.0) + pos.double()
        assert ((got.double() - want).abs() <= rounding(want, t) + want.abs() * 2.0 ** -24).all()
        assert (ops.Embedding(w, ids)[~ok] == 0).all()


def words(kind, tokens, vocab, g):
    if kind == "one":
        return torch.full((tokens,), vocab // 2, dtype=torch.int32, device=DEV)
    if kind == "even":
        return torch.randint(0, vocab, (tokens,), device=DEV, generator=g, dtype=torch.int32)
    u = torch.rand(tokens, device=DEV, generator=g, dtype=torch.float64)
    ids = (torch.exp(u * torch.log(torch.tensor(vocab + 1.0, dtype=torch.float64, device=DEV))).long() - 1).clamp(0, vocab - 1)
    if kind == "padded":
        ids[torch.rand(tokens, device=DEV, generator=g) < 0.4] = -1
        ids[torch.rand(tokens, device=DEV, generator=g) < 0.1] = vocab + 7
    return ids.to(torch.int32)


def grad_check(ids, do, dw, scale, beta):
    vocab, d = dw.shape
    old = dw.clone()
    ok = (ids >= 0) & (ids < vocab)
    at = ids[ok].long()
    rows = do.double().view(-1, d)[ok.view(-1)]
    total = torch.zeros(vocab, d, device=DEV, dtype=torch.float64).index_add_(0, at, rows)
    size = torch.zeros(vocab, d, device=DEV, dtype=torch.float64).index_add_(0, at, rows.abs())
    count = torch.bincount(at, minlength=vocab)
    s = torch.tensor(scale, dtype=F32).double().item()
    want = total * s + (old.double() if beta else 0.0)
    ops.GradEmbedding(ids, do, dw, scale, beta)
    bound = size * abs(s) * count[:, None] * 2.0 ** -24 + want.abs() * 2.0 ** -24 + rounding(want, dw.dtype)
    assert ((dw.double() - want).abs() <= bound).all()
    rest = count == 0
    assert torch.equal(dw[rest], old[rest]) if beta else (dw[rest] == 0).all()


@pytest.mark.parametrize("to,tw", [(F16, F16), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("kind", ["one", "even", "zipf", "padded"])
@pytest.mark.parametrize("tokens,vocab,d", [(1, 1, 1), (7, 3, 8), (33, 600, 40), (700, 513, 513), (2048, 65536, 64), (2049, 1000, 136),
                                            (5000, 70000, 128), (9001, 300, 72), (40000, 300000, 16), (100000, 32000, 24)])
def test_gradient(to, tw, kind, tokens, vocab, d):
    g = gen(tokens)
    ids = words(kind, tokens, vocab, g)
    do = torch.randn(tokens, d, device=DEV, generator=g).to(to)
    dw = torch.randn(vocab, d, device=DEV, generator=g).to(tw)
    grad_check(ids, do, dw, 3.25, 1.0)
    dw.fill_(float("nan"))
    grad_check(ids, do, dw, 0.125, 0.0)


@pytest.mark.parametrize("tokens", [1024, 1025, 2048])
@pytest.mark.parametrize("to,tw", [(F16, F16), (F16, F32), (F32, F32)])
def test_gradient_of_rows_without_wide_accesses(to, tw, tokens):
    for kind in ("one", "padded"):
        test_gradient(to, tw, kind, tokens, 700, 301)


def test_gradient_shapes_pitches_and_nothing_at_all():
    g = gen(9)
    for d in (64, 33):
        buf = torch.full((50, 100), 3.0, device=DEV)
        dw = buf[:, 4:4 + d]
        ids = torch.randint(-2, 52, (4, 25), device=DEV, generator=g, dtype=torch.int32)
        do = torch.randn(4, 25, d, device=DEV, generator=g)
        grad_check(ids, do, dw, 1.0, 1.0)
        grad_check(ids, do, dw, 1.0, 0.0)
        assert (buf[:, :4] == 3).all() and (buf[:, 4 + d:] == 3).all()
    dw = torch.ones(5, 16, device=DEV)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    ops.GradEmbedding(none, torch.empty(0, 16, device=DEV), dw)
    assert (dw == 1).all()
    ops.GradEmbedding(none, torch.empty(0, 16, device=DEV), dw, beta=0.0)
    assert (dw == 0).all()
    assert ops.Embedding(dw, none).shape == (0, 16)


def test_gradient_against_differences():
    g = gen(4)
    w = torch.randn(30, 12, device=DEV, generator=g, dtype=torch.float64)
    ids = torch.randint(0, 30, (50,), device=DEV, generator=g, dtype=torch.int32)
    do = torch.randn(50, 12, device=DEV, generator=g)
    dw = torch.zeros(30, 12, device=DEV)
    ops.GradEmbedding(ids, do, dw, 1.5)
    u = torch.randn(30, 12, device=DEV, generator=g, dtype=torch.float64)

    def value(w):
        return (1.5 * w[ids.long()] * do.double()).sum().item()
    # the operator is linear: the difference quotient is exact up to 64-bit rounding
    assert abs((value(w + 1e-3 * u) - value(w - 1e-3 * u)) / 2e-3 - (dw.double() * u).sum().item()) <= 1e-4 * (dw.double() * u).norm().item()


def test_gradient_repeats_streams_and_capture():
    g = gen(6)
    ids = words("zipf", 20000, 5000, g)
    do = torch.randn(20000, 96, device=DEV, generator=g).half()
    dw = torch.empty(5000, 96, device=DEV).half()
    ops.GradEmbedding(ids, do, dw, 2.0, 0.0)
    first = dw.clone()
    side = torch.cuda.Stream()
    for _ in range(5):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = torch.empty_like(dw)
            ops.GradEmbedding(ids, do, other, 2.0, 0.0)
            row = ops.Embedding(other, ids, 0.5)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, first) and torch.equal(row, ops.Embedding(first, ids, 0.5))
    graphs = []
    for _ in range(2):
        target = torch.zeros_like(dw)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            ops.GradEmbedding(ids, do, target, 2.0, 1.0)
            out = ops.Embedding(target, ids)
        graphs.append((gr, target, out))
    ids.copy_(words("zipf", 20000, 5000, g))
    for gr, target, out in graphs:
        gr.replay()
    want = torch.zeros_like(dw)
    ops.GradEmbedding(ids, do, want, 2.0, 1.0)
    torch.cuda.synchronize()
    for gr, target, out in graphs:
        assert torch.equal(target, want) and torch.equal(out, want[ids.long()])
