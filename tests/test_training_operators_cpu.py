"""Argument checks of the embedding and gradient-clipping entry points; they run before any CUDA call."""
import ctypes

import pytest
import torch

from niutensor_b200 import capi, ops

P = 4096        # an address that is never dereferenced
F16, F32 = capi.X_FLOAT16, capi.X_FLOAT


def rows(ids=P, w=P, pos=P, out=P, dtype=F16, tokens=4, vocab=10, dim=8, ldw=8, ldo=8, pos_rows=2, scale=1.0):
    return capi.lib().ntb_embedding(0, None, ids, w, pos, out, dtype, tokens, vocab, dim, ldw, ldo, pos_rows, scale)


@pytest.mark.parametrize("change,code", [
    (dict(ids=None), capi.ERR_ARG), (dict(w=None), capi.ERR_ARG), (dict(out=None), capi.ERR_ARG), (dict(dtype=capi.X_INT8), capi.ERR_DTYPE),
    (dict(tokens=-1), capi.ERR_ARG), (dict(vocab=-1), capi.ERR_ARG), (dict(ldw=7), capi.ERR_ARG), (dict(ldo=4), capi.ERR_ARG),
    (dict(pos_rows=0), capi.ERR_ARG), (dict(tokens=0, ids=None), capi.OK), (dict(dim=0), capi.OK),
])
def test_embedding_refuses(change, code):
    assert rows(**change) == code


def grad(ids=P, do=P, dw=P, to=F16, tw=F32, tokens=4, vocab=10, dim=8, ldo=8, ldw=8, scale=1.0, beta=1.0, work=P, bytes_=None):
    lib = capi.lib()
    return lib.ntb_embedding_grad(0, None, ids, do, dw, to, tw, tokens, vocab, dim, ldo, ldw, scale, beta, work,
                                  lib.ntb_embedding_grad_work(4, 8) if bytes_ is None else bytes_)


@pytest.mark.parametrize("change,code", [
    (dict(ids=None), capi.ERR_ARG), (dict(do=None), capi.ERR_ARG), (dict(dw=None), capi.ERR_ARG), (dict(work=None), capi.ERR_ARG),
    (dict(work=P + 8), capi.ERR_ARG), (dict(bytes_=8), capi.ERR_ARG), (dict(beta=0.5), capi.ERR_ARG), (dict(beta=float("nan")), capi.ERR_ARG),
    (dict(to=F32, tw=F16), capi.ERR_DTYPE), (dict(to=capi.X_DOUBLE), capi.ERR_DTYPE), (dict(ldo=7), capi.ERR_ARG), (dict(ldw=0), capi.ERR_ARG),
    (dict(dim=-1), capi.ERR_ARG), (dict(vocab=0), capi.OK), (dict(tokens=0, ids=None, do=None), capi.OK), (dict(vocab=2 ** 31 - 1), capi.ERR_LIMIT),
])
def test_embedding_gradient_refuses(change, code):
    assert grad(**change) == code


def clip(count=2, grads=(P, P), out=(P, P), types=(F32, F16), counts=(4, 4), max_norm=1.0, norm=P, work=P, bytes_=None):
    lib = capi.lib()
    n = max(1, count)
    return lib.ntb_clip_grad_norm(0, None, count, (ctypes.c_void_p * n)(*grads[:n]), (ctypes.c_void_p * n)(*out[:n]), (ctypes.c_int * n)(*types[:n]),
                                  (ctypes.c_longlong * n)(*counts[:n]), max_norm, norm, work,
                                  lib.ntb_clip_grad_norm_work(count) if bytes_ is None else bytes_)


@pytest.mark.parametrize("change,code", [
    (dict(count=-1), capi.ERR_ARG), (dict(norm=None), capi.ERR_ARG), (dict(work=None), capi.ERR_ARG), (dict(work=P + 4), capi.ERR_ARG),
    (dict(bytes_=8), capi.ERR_ARG), (dict(max_norm=-0.1), capi.ERR_ARG), (dict(max_norm=float("nan")), capi.ERR_ARG),
    (dict(grads=(P, None)), capi.ERR_ARG), (dict(out=(None, P)), capi.ERR_ARG), (dict(grads=(P + 2, P)), capi.ERR_ARG),
    (dict(out=(P, P + 1)), capi.ERR_ARG), (dict(types=(F32, capi.X_DOUBLE)), capi.ERR_DTYPE), (dict(counts=(4, -1)), capi.ERR_ARG),
    (dict(counts=(4, 1 << 45)), capi.ERR_LIMIT), (dict(counts=(1 << 44, 1 << 44)), capi.ERR_LIMIT),
])
def test_clip_refuses(change, code):
    assert clip(**change) == code


def test_operators_refuse_host_tensors():
    w, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: ops.Embedding(w, ids), lambda: ops.GradEmbedding(ids, torch.zeros(3, 8), w), lambda: ops.ClipGradNorm([w], 1.0)):
        with pytest.raises(ops.NtError, match="no CPU path"):
            call()
