"""Extents past 32 bits, which a broadcast or a large tensor can have, are refused before anything is made or launched."""
import pytest
import torch

from niutensor_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PAST = 2 ** 32 + 1                # as an int of 32 bits it would read 1


def refused(call):
    held = torch.cuda.memory_allocated()
    with pytest.raises(ops.NtError, match="32 bits"):
        call()
    assert torch.cuda.memory_allocated() == held


@pytest.mark.parametrize("axis", [0, 1])
def test_cross_attention(axis):
    one = torch.zeros(1, 1, 1, 8, device=DEV).half()
    shape = [1, 1, 1, 8]
    shape[axis] = PAST
    x = one.expand(shape)
    refused(lambda: ops.CrossAttention(x, x, x))
    if axis == 1:
        refused(lambda: ops.CrossAttention(x, one, one))
    lse = torch.zeros(1, 1, 1, device=DEV).expand(shape[:3])
    refused(lambda: ops.GradCrossAttention(x, x, x, x, lse, x))


def test_embedding_rows_and_gradient():
    ids = torch.zeros(PAST, dtype=torch.int32, device=DEV)
    w = torch.zeros(4, 1, device=DEV).half()
    refused(lambda: ops.Embedding(w, ids))
    dout = torch.zeros(PAST, 1, device=DEV).half()
    refused(lambda: ops.GradEmbedding(ids, dout, w))
    del dout, ids
    few = torch.zeros(3, dtype=torch.int32, device=DEV)
    wide = torch.zeros(PAST, 1, device=DEV).half()
    refused(lambda: ops.Embedding(wide, few))
    refused(lambda: ops.GradEmbedding(few, torch.zeros(3, 1, device=DEV).half(), wide))
    refused(lambda: ops.Embedding(wide.t(), few))
