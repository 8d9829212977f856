"""Argument checks of the cross-attention entry points; they run before any CUDA call."""
import ctypes

import pytest
import torch

from niutensor_b200 import capi, ops

P = 4096        # an address that is never dereferenced


def layouts(n, d=64, length=32, heads=4, **change):
    out = []
    for i in range(n):
        one = dict(batch=heads * length * d, head=length * d, row=d)
        one.update(change.get("t%d" % i, {}))
        out.append(capi.HeadsLayout(**one))
    return (capi.HeadsLayout * n)(*out)


def forward(q=P, k=P, v=P, out=P, dtype=capi.X_FLOAT16, batch=2, heads=4, kv=4, n=32, m=32, d=64, lay=None, scale=0.125):
    return capi.lib().ntb_cross_attention(0, None, q, k, v, out, None, dtype, batch, heads, kv, n, m, d,
                                          lay if lay is not None else layouts(4), None, None, scale)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), capi.ERR_ARG), (dict(k=None), capi.ERR_ARG), (dict(v=None), capi.ERR_ARG), (dict(out=None), capi.ERR_ARG),
    (dict(dtype=capi.X_FLOAT), capi.ERR_DTYPE), (dict(dtype=capi.X_INT8), capi.ERR_DTYPE),
    (dict(batch=-1), capi.ERR_ARG), (dict(n=-1), capi.ERR_ARG), (dict(m=-2), capi.ERR_ARG),
    (dict(heads=6), capi.ERR_SHAPE), (dict(kv=0), capi.ERR_SHAPE),
    (dict(d=60), capi.ERR_LIMIT), (dict(d=0), capi.ERR_LIMIT), (dict(d=136), capi.ERR_LIMIT),
    (dict(scale=0.0), capi.ERR_ARG), (dict(scale=-1.0), capi.ERR_ARG), (dict(scale=float("inf")), capi.ERR_ARG),
    (dict(scale=float("nan")), capi.ERR_ARG),
    (dict(q=P + 8), capi.ERR_ARG), (dict(v=P + 2), capi.ERR_ARG), (dict(out=P + 8), capi.ERR_ARG),
    (dict(lay=layouts(4, t0=dict(row=65))), capi.ERR_ARG), (dict(lay=layouts(4, t1=dict(head=2052))), capi.ERR_ARG),
    (dict(lay=layouts(4, t2=dict(batch=1 << 40))), capi.ERR_ARG), (dict(lay=layouts(4, t1=dict(row=-64))), capi.ERR_ARG),
    (dict(lay=layouts(4, t3=dict(batch=0))), capi.ERR_ARG), (dict(lay=layouts(4, t1=dict(row=0))), capi.ERR_ARG),
])
def test_forward_refuses(change, code):
    assert forward(**change) == code


def test_nothing_to_do_is_no_error():
    assert forward(batch=0) == capi.OK
    assert forward(n=0, q=None, out=None) == capi.OK
    assert forward(heads=0, kv=0) == capi.OK


def test_without_a_device_there_is_no_fallback():
    if not torch.cuda.is_available():
        assert forward() == capi.ERR_CUDA


def test_operator_refuses_host_tensors():
    x = torch.zeros(1, 1, 2, 64, dtype=torch.float16)
    with pytest.raises(ops.NtError, match="no CPU path"):
        ops.CrossAttention(x, x, x)


def test_layout_structure_matches_the_header():
    assert ctypes.sizeof(capi.HeadsLayout) == 24


def grad(q=P, k=P, v=P, out=P, lse=P, dout=P, dq=P, dk=P, dv=P, work=P, bytes_=None, dtype=capi.X_FLOAT16, batch=2, heads=4, kv=4, n=32, m=32,
         d=64, lay=None, scale=0.125):
    lib = capi.lib()
    need = lib.ntb_cross_attention_grad_work(2, 4, 32) if bytes_ is None else bytes_
    return lib.ntb_cross_attention_grad(0, None, q, k, v, out, lse, dout, dq, dk, dv, work, need, dtype, batch, heads, kv, n, m, d,
                                        lay if lay is not None else layouts(8), None, None, scale)


@pytest.mark.parametrize("change,code", [
    (dict(q=None), capi.ERR_ARG), (dict(lse=None), capi.ERR_ARG), (dict(dout=None), capi.ERR_ARG), (dict(dq=None), capi.ERR_ARG),
    (dict(dk=None), capi.ERR_ARG), (dict(dv=None), capi.ERR_ARG), (dict(work=None), capi.ERR_ARG), (dict(work=P + 4), capi.ERR_ARG),
    (dict(bytes_=64), capi.ERR_ARG), (dict(dtype=capi.X_FLOAT), capi.ERR_DTYPE), (dict(kv=3), capi.ERR_SHAPE),
    (dict(d=12), capi.ERR_LIMIT), (dict(scale=0.0), capi.ERR_ARG), (dict(m=-1), capi.ERR_ARG),
    (dict(lay=layouts(8, t4=dict(row=66))), capi.ERR_ARG), (dict(lay=layouts(8, t6=dict(head=0))), capi.ERR_ARG),
    (dict(lay=layouts(8, t7=dict(batch=0))), capi.ERR_ARG), (dict(lay=layouts(8, t5=dict(row=56))), capi.ERR_ARG),
    (dict(dq=P + 2), capi.ERR_ARG),
])
def test_gradient_refuses(change, code):
    assert grad(**change) == code


def test_gradient_work_bytes():
    lib = capi.lib()
    assert lib.ntb_cross_attention_grad_work(2, 4, 1) == 2 * 4 * 1024
    assert lib.ntb_cross_attention_grad_work(1, 1, 129) == 2048
    assert lib.ntb_cross_attention_grad_work(3, 5, 0) == 0 and lib.ntb_cross_attention_grad_work(-1, 5, 9) == 0
    assert lib.ntb_cross_attention_grad_work(1 << 12, 128, 1 << 16) == (1 << 19) * 512 * 1024        # beyond 32 bits
