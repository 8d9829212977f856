"""Lists whose entries overlap: the clipping would write what another part of the call still reads, so they are refused."""
import random

import pytest
import torch

from niutensor_b200 import capi, ops
from tests.test_training_operators_cpu import F16, F32, P, clip

# what an accepted list answers where there is no device; with one these addresses may not be used
NO_DEVICE = capi.ERR_CUDA


def plain(n, size=4, step=16):
    return tuple(P + i * step for i in range(n)), (F32,) * n, (size,) * n


@pytest.mark.parametrize("change", [
    dict(grads=(P, P + 64), out=(P + 64, P)),                                      # swapped
    dict(grads=(P, P + 64), out=(P + 64, P + 128)),                                # shifted by an entry
    dict(grads=(P, P + 64), out=(P + 4, P + 64)),                                  # shifted by an element
    dict(grads=(P + 4, P + 64), out=(P, P + 64)),
    dict(grads=(P, P + 64), out=(P + 128, P + 128)),                               # one target twice
    dict(grads=(P, P + 64), out=(P + 128, P + 136)),                               # targets that overlap in part
    dict(grads=(P, P + 8), out=(P, P + 8)),                                        # in place, overlapping in part
    dict(grads=(P, P), out=(P, P)),
    dict(grads=(P, P + 14), out=(P, P + 14), types=(F32, F16)),
    dict(grads=(P, P + 256), out=(P + 512, P + 300), counts=(4, 64)),              # a target inside a long source
    dict(grads=(P + 300, P + 1024), out=(P, P + 512), counts=(4, 64), types=(F32, F32)) | dict(out=(P + 2048, P + 256)),
])
def test_overlaps_are_refused(change):
    assert clip(**change) == capi.ERR_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")
@pytest.mark.parametrize("change", [
    dict(grads=(P, P + 16), out=(P, P + 16)), dict(grads=(P + 16, P), out=(P + 16, P)),          # neighbours, in any order
    dict(grads=(P, P + 16), out=(P + 32, P + 48)), dict(grads=(P, P), out=(P + 32, P + 48)),       # a source may be read twice
    dict(grads=(P, P + 16), out=(P + 32, P + 16)),                                                  # one of them in place
    dict(grads=(P, None), out=(P, None), counts=(4, 0)), dict(grads=(P, P), out=(P, P), counts=(4, 0)),
])
def test_others_are_not(change):
    assert clip(**change) == NO_DEVICE


@pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are made up")
@pytest.mark.parametrize("n", [65, 500])
def test_long_lists_against_every_pair(n):
    rng = random.Random(n)
    for _ in range(20):
        spread = rng.choice([40 * n, 4000 * n])
        grads = [P + 4 * rng.randrange(spread) for _ in range(n)]
        out = [g if rng.random() < 0.5 else P + 4 * rng.randrange(spread) for g in grads]
        counts = [rng.choice([0, 1, 3, 9]) for _ in range(n)]

        def hit(a, i, b, j):
            return counts[i] and counts[j] and a < b + 4 * counts[j] and b < a + 4 * counts[i]
        wrong = any(hit(out[i], i, out[j], j) for i in range(n) for j in range(i)) or \
            any(hit(grads[i], i, out[j], j) for i in range(n) if grads[i] != out[i] for j in range(n))
        got = clip(count=n, grads=grads, out=out, types=(F32,) * n, counts=counts)
        assert got == (capi.ERR_ARG if wrong else NO_DEVICE)


@pytest.mark.gpu
def test_the_operator_refuses_them():
    a, b, c = (torch.ones(100, device="cuda:0") for _ in range(3))
    pool = torch.ones(300, device="cuda:0")
    for grads, out in (([a, b], [b, a]), ([a, b], [b, c]), ([pool[:100], pool[50:150]], None), ([pool[:100]], [pool[1:101]]), ([a], [a[1:]])):
        before = [x.clone() for x in grads]
        with pytest.raises(ops.NtError):
            ops.ClipGradNorm(grads, 0.5, out=out)
        for x, y in zip(grads, before):
            assert torch.equal(x, y)
    ops.ClipGradNorm([a, b], 0.5, out=[c, b])
    ops.ClipGradNorm([pool[:100], pool[100:200]], 0.5)
    ops.ClipGradNorm([pool[100:200], pool[:100]], 0.5, out=[a, b])
