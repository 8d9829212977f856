"""Clipping by factors below a float's normal range: the norm is within 2^-21 and the factor, of which a power of two is taken
out, within 2^-24 of itself; the product with that power is exact where the result is normal, and the last product rounds
once (2^-24, below the normal range 2^-149 at most)."""
import math

import pytest
import torch

from niutensor_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [5, 4097])
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("max_norm", [1.0, 1.0e-3, 1.0e-8, 1.0e-30, 1.0e-38])
def test_tiny_factors(n, shift, max_norm):
    g = torch.Generator(device="cuda:0").manual_seed(1)
    pool = torch.randn(n + shift, device="cuda:0", generator=g)
    x = pool[shift:]
    x *= 2.0e38 / x.norm()
    before, halves = x.double(), torch.full((9,), 3.0, device="cuda:0").half()
    want = math.sqrt((before ** 2).sum().item())
    top = torch.tensor(max_norm, dtype=torch.float32).double().item()
    out = torch.empty(n + 2, device="cuda:0")[2:]
    assert abs(ops.ClipGradNorm([x, halves], max_norm, out=[out, torch.empty_like(halves)]).item() - want) <= want * 2.0 ** -21
    ops.ClipGradNorm([x, halves], max_norm)
    ref = before * (top / want)
    bound = ref.abs() * 2.0 ** -20 + 2.0 ** -149
    assert ((x.double() - ref).abs() <= bound).all() and torch.equal(out, x) and (halves == 0).all()
