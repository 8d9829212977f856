"""The norm of a list of gradients and their clipping, against 64-bit sums.

The norm: fp64 partial sums (halves: eight exact products summed in fp32, 2^-21 at most), rounded to fp32 once:
within 2^-21 of itself. A clipped element: the factor is rounded to fp32 (2^-24), the product once more (2^-24) and
to its type (2^-11, at most 2^-25, for halves; for floats the product is the result, at most 2^-149)."""
import math

import pytest
import torch

from niutensor_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(sizes, types, scale=0.1, seed=1, shift=0):
    """tensors one behind the other in a pool, `shift` elements off its start"""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = types[i % len(types)]
        count = math.prod(n) if isinstance(n, tuple) else n
        pool = (torch.randn(count + shift, device=DEV, generator=g) * scale).to(t)
        x = pool[shift:]
        out.append(x.view(n) if isinstance(n, tuple) else x)
    return out


def norm_of(grads):
    return math.sqrt(math.fsum((x.double() ** 2).sum().item() for x in grads))


def check(grads, max_norm, out=None):
    before = [x.clone() for x in grads]
    want = norm_of(before)
    norm = ops.ClipGradNorm(grads, max_norm, out=out)
    assert norm.dtype == torch.float32 and norm.shape == ()
    if math.isinf(want):                                 # an infinity among the values: reported, nothing changed
        assert math.isinf(norm.item())
        for b, o in zip(before, grads if out is None else out):
            assert torch.equal(o, b)
        return
    assert abs(norm.item() - want) <= want * 2.0 ** -21
    f = max_norm / want if want > max_norm else 1.0
    for x, b, o in zip(grads, before, grads if out is None else out):
        ref = b.double() * f
        bound = ref.abs() * 2.0 ** -20 + (ref.abs() * 2.0 ** -11 + 2.0 ** -25 if x.dtype == torch.float16 else 2.0 ** -149)
        assert ((o.double() - ref).abs() <= bound).all()
        if want <= max_norm:
            assert torch.equal(o, b)
        if out is not None:
            assert torch.equal(x, b)


F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("types", [[F16], [F32], [F16, F32]])
@pytest.mark.parametrize("sizes", [[1], [7, 3, 1], [(512, 512), (512,), (512, 2048), (2048,), (1,)], [8192, 16384, 16385, 8191, 40000],
                                   [0, 5, 0, 0, 100000, 0], [3] * 64, [17] * 65, [129, 1000] * 700, [3000001]])
def test_clipped_and_not(types, sizes):
    for shift in (0, 1, 3):
        check(make(sizes, types, shift=shift), 0.05)
        check(make(sizes, types, shift=shift), 1.0e6)
        grads = make(sizes, types, shift=shift)
        check(grads, 0.05, out=[torch.full_like(x, 9.0) for x in grads])
        check(grads, 1.0e6, out=[torch.full_like(x, 9.0) for x in grads])


def test_other_alignment_in_and_out():
    grads = make([1000, 33333], [F16, F32], shift=1)
    check(grads, 0.5, out=[torch.empty(x.numel() + 2, dtype=x.dtype, device=DEV)[2:] for x in grads])


def test_norms_whose_squares_pass_32_bits():
    check(make([5000], [F32], scale=1.0e25), 1.0)
    grads = make([5000], [F32], scale=1.0e-30)
    check(grads, 1.0e-29)
    check(make([5000], [F16], scale=3.0e4), 1.0)         # some values are infinite as halves
    check([x.clamp(-65504, 65504) for x in make([5000], [F16], scale=3.0e4)], 1.0)
    check(make([5000], [F16], scale=2.0 ** -22), 2.0 ** -20)


def test_not_finite_and_nothing():
    for bad in (float("inf"), float("nan")):
        grads = make([100, 200], [F32, F16])
        grads[1][3] = bad
        before = [x.clone() for x in grads]
        norm = ops.ClipGradNorm(grads, 0.1)
        assert math.isinf(norm.item()) if math.isinf(bad) else math.isnan(norm.item())
        out = [torch.zeros_like(x) for x in grads]
        ops.ClipGradNorm(grads, 0.1, out=out)
        for x, b, o in zip(grads, before, out):
            assert torch.equal(x.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0)) and torch.equal(o.nan_to_num(nan=7.0), b.nan_to_num(nan=7.0))
    grads = make([50], [F32])
    ops.ClipGradNorm(grads, 0.0)
    assert (grads[0] == 0).all()
    check(make([50], [F32]), float("inf"))
    zero = [torch.zeros(10, device=DEV)]
    assert ops.ClipGradNorm(zero, 1.0).item() == 0.0 and (zero[0] == 0).all()
    assert ops.ClipGradNorm([torch.empty(0, device=DEV)], 1.0).item() == 0.0


def test_refusals():
    x = torch.ones(4, device=DEV)
    for call in (lambda: ops.ClipGradNorm([], 1.0), lambda: ops.ClipGradNorm([x, x], 1.0), lambda: ops.ClipGradNorm([x], -1.0),
                 lambda: ops.ClipGradNorm([x], float("nan")), lambda: ops.ClipGradNorm([x.double()], 1.0),
                 lambda: ops.ClipGradNorm([x], 1.0, out=[x.half()]), lambda: ops.ClipGradNorm([torch.ones(4, 4, device=DEV).t()[1:]], 1.0),
                 lambda: ops.ClipGradNorm([x.cpu()], 1.0)):
        with pytest.raises(ops.NtError):
            call()


def test_repeats_streams_and_capture():
    grads = make([(300, 300), 7, (64, 1000)] * 3, [F32, F16])
    out = [torch.empty_like(x) for x in grads]
    norm = ops.ClipGradNorm(grads, 0.3, out=out)
    first = [norm.clone()] + [x.clone() for x in out]
    side = torch.cuda.Stream()
    for _ in range(4):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = [torch.empty_like(x) for x in grads]
            n = ops.ClipGradNorm(grads, 0.3, out=again)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip([n] + again, first):
            assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        res = [torch.empty_like(x) for x in grads]
        with torch.cuda.graph(g):
            n = ops.ClipGradNorm(grads, 0.3, out=res)
        graphs.append((g, [n] + res))
    for x in grads:
        x.mul_(2.0)
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = [torch.empty_like(x) for x in grads]
    n = ops.ClipGradNorm(grads, 0.3, out=want)
    for _, res in graphs:
        for a, b in zip(res, [n] + want):
            assert torch.equal(a, b)


def test_a_norm_past_a_float():
    """it reads as infinite, so the values stay as they are"""
    x = torch.full((5,), 3.0e38, device=DEV)
    out = torch.empty_like(x)
    assert math.isinf(ops.ClipGradNorm([x], 1.0, out=[out]).item()) and torch.equal(out, x)
    assert math.isinf(ops.ClipGradNorm([x], 1.0).item()) and (x == 3.0e38).all()
