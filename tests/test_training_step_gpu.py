"""The operators of a training step as they are used together: a decoder sublayer over an encoder's states, from
token ids to clipped gradients, against the same step in 64 bits; and a decoding step."""
import math

import pytest
import torch

from niutensor_b200 import capi, ops
from niutensor_b200.capi import X_NOTRANS, X_TRANS

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
B, H, N, M, D, VOCAB = 3, 4, 37, 50, 64, 500
WIDTH = H * D


def heads(x, length):
    return x.view(B, length, H, D).transpose(1, 2)


def setup(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def rand(*shape, s=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * s).half()
    w = dict(emb=rand(VOCAB, WIDTH, s=WIDTH ** -0.5), q=rand(WIDTH, WIDTH, s=WIDTH ** -0.5), k=rand(WIDTH, WIDTH, s=WIDTH ** -0.5),
             v=rand(WIDTH, WIDTH, s=WIDTH ** -0.5))
    enc = rand(B, M, WIDTH)
    pos = rand(N, WIDTH)
    nq, nk = [37, 20, 1], [50, 13, 31]
    ids = torch.randint(0, VOCAB, (B, N), device=DEV, generator=g, dtype=torch.int32)
    for b in range(B):
        ids[b, nq[b]:] = -1
    dout = rand(B, N, WIDTH, s=0.1)
    lens = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (nq, nk)]
    return w, enc, pos, ids, dout, lens


def step(w, enc, pos, ids, dout, lens, max_norm):
    """forward, backward and clipping with the library; gradients of emb, q, k, v, the norm, and the output"""
    nq, nk = lens
    x = ops.Embedding(w["emb"], ids, math.sqrt(WIDTH), pos)
    q, k, v = ops.MMul(x, w["q"]), ops.MMul(enc, w["k"]), ops.MMul(enc, w["v"])
    qh, kh, vh = heads(q, N), heads(k, M), heads(v, M)
    out, lse = ops.CrossAttention(qh, kh, vh, nq, nk, with_lse=True)
    dq, dk, dv = ops.GradCrossAttention(qh, kh, vh, out, lse, heads(dout, N), nq, nk)
    grads = {n: torch.zeros_like(t) for n, t in w.items()}
    dx = torch.zeros_like(x)
    # gradients keep their operands' order of dimensions: merging the heads is a view
    flat = [t.transpose(1, 2).reshape(-1, WIDTH) for t in (dq, dk, dv)]
    assert flat[0].data_ptr() == dq.data_ptr()
    ops.GradMatrixMul(x.view(-1, WIDTH), X_NOTRANS, w["q"], X_NOTRANS, flat[0], dx.view(-1, WIDTH), grads["q"])
    ops.GradMatrixMul(enc.view(-1, WIDTH), X_NOTRANS, w["k"], X_NOTRANS, flat[1], None, grads["k"])
    ops.GradMatrixMul(enc.view(-1, WIDTH), X_NOTRANS, w["v"], X_NOTRANS, flat[2], None, grads["v"])
    ops.GradEmbedding(ids, dx, grads["emb"], math.sqrt(WIDTH))
    norm = ops.ClipGradNorm(list(grads.values()), max_norm)
    return out, grads, norm


def reference(w, enc, pos, ids, dout, lens, max_norm):
    nq, nk = lens
    p = {n: t.double().requires_grad_() for n, t in w.items()}
    word = (ids >= 0)[..., None]
    x = p["emb"][ids.clamp(min=0).long()].masked_fill(~word, 0.0) * math.sqrt(WIDTH) + pos.double()
    q, k, v = heads(x @ p["q"], N), heads(enc.double() @ p["k"], M), heads(enc.double() @ p["v"], M)
    s = (q @ k.transpose(2, 3) / math.sqrt(D)).masked_fill((torch.arange(M, device=DEV)[None] >= nk[:, None])[:, None, None], float("-inf"))
    out = (torch.softmax(s, -1) @ v).masked_fill((torch.arange(N, device=DEV)[None] >= nq[:, None])[:, None, :, None], 0.0)
    (out * heads(dout, N).double()).sum().backward()
    norm = math.sqrt(sum((t.grad ** 2).sum().item() for t in p.values()))
    f = min(1.0, max_norm / norm)
    return out, {n: t.grad * f for n, t in p.items()}, norm


def test_training_step_against_64_bits():
    args = setup(1)
    for max_norm in (1.0e9, 0.5):
        out, grads, norm = step(*args, max_norm)
        want, wgrads, wnorm = reference(*args, max_norm)
        # each result passes through at most six halves on its way (embedding, projection, attention and its
        # weights, gradient, product), each off by up to 2^-11 of what it holds; errors of one value's terms are
        # independent, so the 2-norm of a whole result grows by less than six of them
        bound = 6 * 2.0 ** -11
        assert (out.double() - want).norm() <= bound * want.norm()
        for n in grads:
            assert (grads[n].double() - wgrads[n]).norm() <= bound * wgrads[n].norm(), n
        assert abs(norm.item() - wnorm) <= bound * wnorm
    assert capi.lib().ntb_device_status(0) == capi.OK


def test_training_step_captured_beside_an_eager_one():
    """one graph of the whole step, replayed on new data while eager steps run before and after it"""
    args = setup(2)
    first = step(*args, 0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads, norm = step(*args, 0.5)
    w, enc, pos, ids, dout, lens = args
    new = setup(3)
    for a, b in zip((enc, pos, ids, dout, *lens, *w.values()), (new[1], new[2], new[3], new[4], *new[5], *new[0].values())):
        a.copy_(b)
    eager = step(*args, 0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager[0]) and torch.equal(norm, eager[2])
    for n in grads:
        assert torch.equal(grads[n], eager[1][n]), n
    assert not torch.equal(first[0], eager[0])


def test_decoding_step_of_a_beam():
    """hypotheses of a sentence as rows of one call over its states equal one call a hypothesis"""
    w, enc, pos, ids, dout, (nq, nk) = setup(4)
    beams = 5
    k, v = heads(ops.MMul(enc, w["k"]), M), heads(ops.MMul(enc, w["v"]), M)
    tokens = torch.randint(0, VOCAB, (B, beams), device=DEV, dtype=torch.int32)
    x = ops.Embedding(w["emb"], tokens, math.sqrt(WIDTH), pos[7:8])
    q = ops.MMul(x, w["q"]).view(B, beams, H, D).transpose(1, 2)
    out = ops.CrossAttention(q, k, v, None, nk)
    for i in range(beams):
        one = ops.CrossAttention(q[:, :, i:i + 1], k, v, None, nk)
        assert (out[:, :, i:i + 1].double() - one.double()).abs().max() <= 2.0 ** -10 * one.double().abs().max()
    merged = out.transpose(1, 2).reshape(B, beams, WIDTH)
    assert merged.data_ptr() == out.data_ptr()
    want = torch.softmax((q.double() @ k.double().transpose(2, 3) / 8.0).masked_fill(
        (torch.arange(M, device=DEV)[None] >= nk[:, None])[:, None, None], float("-inf")), -1) @ v.double()
    assert (out.double() - want).norm() <= 2.0 ** -10 * want.norm()
