"""Embedding rows and their gradient at the ends of 32-bit sizes: what the kernels' indices cannot reach is refused, the
rest is right."""
import pytest
import torch

from niutensor_b200 import capi, ops
from tests.test_training_operators_cpu import F16, F32, grad, rows

BIG = 2 ** 31 - 1


@pytest.mark.parametrize("change", [
    dict(dim=BIG, ldw=BIG, ldo=BIG), dict(dim=BIG - 254, ldw=BIG, ldo=BIG, dtype=F32),
])
def test_rows_past_the_indices_are_refused(change):
    assert rows(**change) == capi.ERR_LIMIT


@pytest.mark.parametrize("change", [
    dict(dim=BIG, ldw=BIG, ldo=BIG), dict(dim=BIG - 254, ldw=BIG, ldo=BIG),                # columns
    dict(dim=1 << 30, ldw=1 << 30, ldo=1 << 30, tokens=2048, to=F32),                      # columns times tokens of one launch
    dict(dim=(1 << 24) + 7, ldw=1 << 25, ldo=1 << 25, tokens=5000),                        # columns of a sorted sum
])
def test_gradients_past_the_indices_are_refused(change):
    assert grad(bytes_=1 << 60, **change) == capi.ERR_LIMIT



@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [5, 3000])
def test_a_vocabulary_that_ends_at_32_bits(tokens):
    """the largest vocabulary: rows that no word has are cleared to the last, the last word's is summed"""
    vocab = BIG - 1
    dw = torch.full((vocab, 1), 9.0, dtype=torch.float16, device="cuda:0")
    ids = torch.full((tokens,), vocab - 1, dtype=torch.int32, device="cuda:0")
    ids[::2] = 7
    dout = torch.ones(tokens, 1, dtype=torch.float16, device="cuda:0")
    ops.GradEmbedding(ids, dout, dw, beta=0.0)
    half = tokens // 2
    assert dw[7].item() == torch.tensor(float(tokens - half)).half().item() and dw[-1].item() == torch.tensor(float(half)).half().item()
    dw[7], dw[-1] = 0, 0
    for lo in range(0, vocab, 1 << 28):
        assert not dw[lo:lo + (1 << 28)].any()
    assert capi.lib().ntb_device_status(0) == capi.OK
