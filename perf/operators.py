"""Cases and plain forms of the operators around an encoder-decoder's training and decoding:
attention of a decoder's positions to an encoder's states (forward, gradients, and the step of
a few new tokens), embedding rows with a scale and their gradient, and the clipping of a list
of gradients to a global norm.

`own` false: elementary torch operations in 32 bits (64 for the long sum of squares), rounded
once at the end. `own` true: the calls a program makes of niutensor_b200.ops. `exact` gives the
operators' definitions in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
HALF, FLOAT = "half", "float"
TYPES = {HALF: torch.float16, FLOAT: torch.float32}


def _attention(name, batch, heads_q, heads_kv, len_q, len_k, dim, ragged, split, lse):
    return {"name": name, "op": "attention", "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv, "len_q": len_q,
            "len_k": len_k, "dim": dim, "ragged": ragged, "split": split, "lse": lse}


def _attention_grad(name, batch, heads_q, heads_kv, len_q, len_k, dim, ragged, split):
    return {"name": name, "op": "attention_grad", "batch": batch, "heads_q": heads_q, "heads_kv": heads_kv, "len_q": len_q,
            "len_k": len_k, "dim": dim, "ragged": ragged, "split": split}


def _embedding(name, op, tokens, length, vocab, dim, dtype):
    return {"name": name, "op": op, "tokens": tokens, "length": length, "vocab": vocab, "dim": dim, "type": dtype}


def _clip(name, layers, width, inner, vocab, dtype):
    return {"name": name, "op": "clip", "layers": layers, "width": width, "inner": inner, "vocab": vocab, "type": dtype}


def listed():
    return [
        # one greedy step for one short sentence: one new token, eight heads of 64; pure latency
        _attention("step_one_sentence", 1, 8, 8, 1, 23, 64, False, False, False),
        # one step over long documents, four query heads to a key head: the states are read once
        _attention("step_long", 8, 32, 8, 1, 16384, 128, True, False, False),
        # training, forward: a padded batch of sentences, heads as the projection lays them out
        _attention("sentences", 64, 8, 8, 61, 73, 64, True, True, True),
        # training, forward: document translation, long on both sides, four heads of 128 to a sentence's four
        _attention("documents", 4, 16, 16, 2000, 8192, 128, False, False, True),
        # training, backward: sentences at the transformer sample's length cap and head size
        _attention_grad("sentences_grad", 64, 4, 4, 200, 200, 128, True, True),
        # training, backward: documents, four query heads share the gradients of a key head
        _attention_grad("documents_grad", 2, 16, 4, 1777, 4100, 128, False, False),
        # one decoding step: the rows of 256 hypotheses out of a large vocabulary
        _embedding("rows_step", "embedding", 256, 1, 65536, 512, HALF),
        # a training batch of tokens, each with its position's row
        _embedding("rows_batch", "embedding", 32768, 256, 32000, 1024, FLOAT),
        # gradient of a batch of sentences into a large vocabulary: most rows stay zero
        _embedding("rows_grad", "embedding_grad", 4096, 64, 65536, 512, HALF),
        # gradient of a large batch: frequent words gather thousands of rows each
        _embedding("rows_grad_batch", "embedding_grad", 100000, 250, 32000, 1024, FLOAT),
        # all gradients of a small encoder-decoder, one layer a side, in halves
        _clip("clip_small", 1, 256, 1024, 8000, HALF),
        # all gradients of an encoder-decoder with six layers a side
        _clip("clip_model", 6, 1024, 4096, 32000, FLOAT),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "attention", "attention", "attention_grad", "attention_grad", "embedding", "embedding_grad", "clip"])
    if op == "step":
        group, kv = rng.choice([(1, 8), (1, 16), (4, 4), (8, 2), (2, 5)])
        dim, beams = rng.choice([64, 128, 128, 40, 96]), rng.choice([1, 1, 2, 4, 5, 8])
        len_k = _log(rng, 5, 32768)
        batch = max(1, min(_log(rng, 1, 128), (1 << 20) // (len_k * kv) or 1))
        c = _attention("", batch, group * kv, kv, beams, len_k, dim, rng.random() < 0.7, rng.random() < 0.5, False)
    elif op == "attention" or op == "attention_grad":
        group, kv = rng.choice([(1, 4), (1, 8), (1, 16), (4, 2), (3, 2)])
        dim = rng.choice([64, 64, 128, 128, 32, 80, 104])
        len_q, len_k = _log(rng, 9, 3000), _log(rng, 2, 8192)
        most = 900000000 if op == "attention" else (1 << 27)
        batch = max(1, min(_log(rng, 1, 96), most // (group * kv * len_q * len_k) or 1))
        ragged, split = rng.random() < 0.7, rng.random() < 0.5
        if op == "attention":
            c = _attention("", batch, group * kv, kv, len_q, len_k, dim, ragged, split, True)
        else:
            c = _attention_grad("", batch, group * kv, kv, len_q, len_k, dim, ragged, split)
    elif op == "embedding" or op == "embedding_grad":
        length = _log(rng, 1, 512)
        tokens = length * max(1, _log(rng, 16, 65536) // length)
        c = _embedding("", op, tokens, length, _log(rng, 500, 65536), rng.choice([256, 300, 512, 513, 768, 1024]),
                       rng.choice([HALF, FLOAT]))
    else:
        width = rng.choice([96, 129, 256, 512, 640, 1000])
        c = _clip("", rng.randint(1, 6), width, 4 * width, _log(rng, 1000, 32000), rng.choice([HALF, FLOAT]))
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs

def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _lengths(n, longest, g):
    """n lengths spread evenly over the upper half of 1..longest, in an order of their own: their sum is
    the case's, not the seed's"""
    spread = torch.linspace(max(1, longest // 2), longest, n).round().to(torch.int32).to(DEV)
    return spread[torch.randperm(n, generator=g, device=DEV)].contiguous()


def _heads(batch, heads, length, dim, split, g, scale=1.0):
    """[batch, heads, length, dim]: packed, or (split) as a projection's [batch, length, heads * dim] seen by head"""
    shape = (batch, length, heads, dim) if split else (batch, heads, length, dim)
    x = (torch.randn(shape, device=DEV, generator=g) * scale).half()
    return x.transpose(1, 2) if split else x


def _tokens(n, vocab, g):
    """word frequencies fall with the rank as 1 / rank"""
    u = torch.rand(n, device=DEV, generator=g, dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1.0)).long() - 1).clamp_(0, vocab - 1).to(torch.int32)


def _model_shapes(case):
    """the parameters of an encoder-decoder: matrices, their biases and the normalisations' vectors"""
    d, f = case["width"], case["inner"]
    layer = [(d, d), (d,)] * 4 + [(d, f), (f,), (f, d), (d,)] + [(d,)] * 4
    cross = [(d, d), (d,)] * 4 + [(d,)] * 2
    return [(case["vocab"], d)] + layer * case["layers"] + (layer + cross) * case["layers"]


def _pieces(pool, case):
    shapes = _model_shapes(case)
    return [x.view(shape) for x, shape in zip(torch.split(pool, [math.prod(x) for x in shapes]), shapes)]


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["op"] in ("attention", "attention_grad"):
        b, n, m, dim, split = case["batch"], case["len_q"], case["len_k"], case["dim"], case["split"]
        s["q"] = _heads(b, case["heads_q"], n, dim, split, g)
        s["k"] = _heads(b, case["heads_kv"], m, dim, split, g)
        s["v"] = _heads(b, case["heads_kv"], m, dim, split, g)
        s["len_q"] = _lengths(b, n, g) if case["ragged"] and n > 8 else None       # the beams of a step are never padded
        s["len_k"] = _lengths(b, m, g) if case["ragged"] else None
        s["scale"] = 1.0 / math.sqrt(dim)
        if case["op"] == "attention_grad":
            # what the forward pass kept, and the gradient that arrives (of a scaled loss)
            s["out"], s["lse"] = _plain_attention(s)
            s["dout"] = _heads(b, case["heads_q"], n, dim, split, g, 0.25)
    elif case["op"] in ("embedding", "embedding_grad"):
        t = TYPES[case["type"]]
        s["ids"] = _tokens(case["tokens"], case["vocab"], g)
        s["scale"] = math.sqrt(case["dim"])
        if case["op"] == "embedding":
            s["w"] = (torch.randn(case["vocab"], case["dim"], device=DEV, generator=g) / math.sqrt(case["dim"])).to(t)
            s["pos"] = torch.randn(case["length"], case["dim"], device=DEV, generator=g).to(t)
        else:
            s["dout"] = (torch.randn(case["tokens"], case["dim"], device=DEV, generator=g) * 0.1).to(t)
            s["dw"] = torch.empty(case["vocab"], case["dim"], device=DEV, dtype=t)
    else:
        t = TYPES[case["type"]]
        # a pool of gradients, one behind the other as the parameters lie, and a pool for the clipped ones
        s["pool"] = (torch.randn(sum(math.prod(x) for x in _model_shapes(case)), device=DEV, generator=g) * 0.02).to(t)
        s["clipped_pool"] = torch.empty_like(s["pool"])
        s["grads"], s["clipped"] = _pieces(s["pool"], case), _pieces(s["clipped_pool"], case)
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from niutensor_b200 import ops
    case = s["case"]
    if case["op"] == "attention":
        r = ops.CrossAttention(s["q"], s["k"], s["v"], s["len_q"], s["len_k"], scale=s["scale"], with_lse=case["lse"])
        return list(r) if case["lse"] else [r]
    if case["op"] == "attention_grad":
        return list(ops.GradCrossAttention(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["len_q"], s["len_k"],
                                           scale=s["scale"]))
    if case["op"] == "embedding":
        return [ops.Embedding(s["w"], s["ids"], s["scale"], s["pos"])]
    if case["op"] == "embedding_grad":
        ops.GradEmbedding(s["ids"], s["dout"], s["dw"], s["scale"], beta=0.0)
        return [s["dw"]]
    return [ops.ClipGradNorm(s["grads"], 1.0, out=s["clipped"]), s["clipped_pool"]]


def _plain(s):
    case = s["case"]
    if case["op"] == "attention":
        out, lse = _plain_attention(s)
        return [out, lse] if case["lse"] else [out]
    if case["op"] == "attention_grad":
        return _plain_attention_grad(s)
    if case["op"] == "embedding":
        rows = s["w"][s["ids"].long()].float() * s["scale"]
        at = torch.arange(case["tokens"], device=DEV) % case["length"]
        return [(rows + s["pos"][at].float()).to(s["w"].dtype)]
    if case["op"] == "embedding_grad":
        acc = torch.zeros(case["vocab"], case["dim"], device=DEV, dtype=torch.float32)
        acc.index_add_(0, s["ids"].long(), s["dout"].float())
        s["dw"].copy_(acc * s["scale"])
        return [s["dw"]]
    total = torch.zeros((), device=DEV, dtype=torch.float64)
    for x in s["grads"]:
        total = total + (x.double() * x.double()).sum()
    norm = torch.sqrt(total)
    factor = torch.where((norm > 1.0) & torch.isfinite(norm), 1.0 / norm, torch.ones_like(norm)).float()
    for x, y in zip(s["grads"], s["clipped"]):
        y.copy_(x.float() * factor)
    return [norm.float(), s["clipped_pool"]]


def _scores(s):
    """scores by key head, [batch, heads_kv, group * len_q, len_k], the keys past a sentence's end at -inf, and the
    query rows past its end, [batch, 1, 1, len_q, 1], or None"""
    case = s["case"]
    b, kv, n, m = case["batch"], case["heads_kv"], case["len_q"], case["len_k"]
    group = case["heads_q"] // kv
    q = s["q"].float().reshape(b, kv, group * n, case["dim"])
    x = torch.matmul(q, s["k"].float().transpose(2, 3)) * s["scale"]
    if s["len_k"] is not None:
        past = torch.arange(m, device=DEV)[None, :] >= s["len_k"][:, None]
        x.masked_fill_(past[:, None, None, :], float("-inf"))
    rows = None
    if s["len_q"] is not None:
        rows = (torch.arange(n, device=DEV)[None, :] >= s["len_q"][:, None])[:, None, None, :, None]
    return q, x, rows


def _plain_attention(s):
    case = s["case"]
    b, h, kv, n = case["batch"], case["heads_q"], case["heads_kv"], case["len_q"]
    _, x, rows = _scores(s)
    top = x.amax(dim=-1, keepdim=True)
    x = torch.exp(x - top)
    total = x.sum(dim=-1, keepdim=True)
    out = (torch.matmul(x, s["v"].float()) / total).view(b, kv, h // kv, n, case["dim"])
    lse = (top + torch.log(total)).view(b, kv, h // kv, n, 1)
    if rows is not None:
        out = out.masked_fill(rows, 0.0)
        lse = lse.masked_fill(rows, float("-inf"))
    return out.reshape(b, h, n, case["dim"]).half(), lse.reshape(b, h, n)


def _plain_attention_grad(s):
    case = s["case"]
    b, h, kv, n, dim = case["batch"], case["heads_q"], case["heads_kv"], case["len_q"], case["dim"]
    q, x, rows = _scores(s)
    p = torch.exp(x - x.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    dout = s["dout"].float().reshape(b, kv, h // kv, n, dim)
    if rows is not None:
        dout = dout.masked_fill(rows, 0.0)
    dout = dout.view(b, kv, (h // kv) * n, dim)
    dv = torch.matmul(p.transpose(2, 3), dout)
    dp = torch.matmul(dout, s["v"].float().transpose(2, 3))
    ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) * s["scale"]
    dq = torch.matmul(ds, s["k"].float()).view(b, h, n, dim)
    dk = torch.matmul(ds.transpose(2, 3), q)
    return [dq.half(), dk.half(), dv.half()]


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        out, lse, _, _, _ = _exact_attention(s, False)
        return [out, lse] if case["lse"] else [out]
    if case["op"] == "attention_grad":
        return list(_exact_attention(s, True)[2:])
    if case["op"] == "embedding":
        w, pos = s["w"].double(), s["pos"].double()
        sentences = s["ids"].long().view(-1, case["length"])
        return [torch.stack([w[row] * s["scale"] + pos for row in sentences]).view(case["tokens"], case["dim"])]
    if case["op"] == "embedding_grad":
        order = torch.argsort(s["ids"].long(), stable=True)
        sums = torch.cumsum(s["dout"].double()[order], dim=0)
        sums = torch.cat([torch.zeros(1, case["dim"], device=DEV, dtype=torch.float64), sums])
        ends = torch.searchsorted(s["ids"].long()[order], torch.arange(case["vocab"] + 1, device=DEV))
        return [(sums[ends[1:]] - sums[ends[:-1]]) * s["scale"]]
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(x.double())) ** 2 for x in s["grads"]))
    factor = 1.0 / norm if norm > 1.0 else 1.0
    return [torch.tensor(norm, dtype=torch.float64), s["pool"].double() * factor]


def _exact_attention(s, gradients):
    """one sentence and head at a time, over the keys and queries that exist"""
    case = s["case"]
    b, h, kv, dim, scale = case["batch"], case["heads_q"], case["heads_kv"], case["dim"], s["scale"]
    wide = dict(device=DEV, dtype=torch.float64)
    out = torch.zeros(b, h, case["len_q"], dim, **wide)
    lse = torch.full((b, h, case["len_q"]), float("-inf"), **wide)
    dq = torch.zeros_like(out)
    dk = torch.zeros(b, kv, case["len_k"], dim, **wide)
    dv = torch.zeros_like(dk)
    nq = [case["len_q"]] * b if s["len_q"] is None else s["len_q"].tolist()
    nk = [case["len_k"]] * b if s["len_k"] is None else s["len_k"].tolist()
    for i in range(b):
        for j in range(h):
            z = j // (h // kv)
            q = s["q"][i, j, :nq[i]].double()
            k, v = s["k"][i, z, :nk[i]].double(), s["v"][i, z, :nk[i]].double()
            x = (q @ k.T) * scale
            total = torch.logsumexp(x, dim=1)
            p = torch.exp(x - total[:, None])
            o = p @ v
            if not gradients:
                out[i, j, :nq[i]], lse[i, j, :nq[i]] = o, total
                continue
            do = s["dout"][i, j, :nq[i]].double()
            dv[i, z, :nk[i]] += p.T @ do
            dx = p * (do @ v.T - (do * o).sum(dim=1, keepdim=True))
            dq[i, j, :nq[i]] = (dx @ k) * scale
            dk[i, z, :nk[i]] += (dx.T @ q) * scale
    return out, lse, dq, dk, dv


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["op"] in ("attention", "attention_grad"):
        b, h, kv, n, m, d = (case[x] for x in ("batch", "heads_q", "heads_kv", "len_q", "len_k", "dim"))
        # lengths are spread over the upper half of their range
        mean_n = n * 0.75 if case["ragged"] and n > 8 else n
        mean_m = m * 0.75 if case["ragged"] else m
        rows, keys = b * h * mean_n * d * 2, b * kv * mean_m * d * 2
        product = 2.0 * b * h * mean_n * mean_m * d
        if case["op"] == "attention":
            return {"bytes": int(2 * rows + 2 * keys + (4 * b * h * mean_n if case["lse"] else 0)), "flops": int(2 * product)}
        # five products: scores, the gradients of the probabilities, and those of v, k and q
        return {"bytes": int(4 * rows + 4 * keys + 4 * b * h * mean_n), "flops": int(5 * product)}
    if case["op"] in ("embedding", "embedding_grad"):
        size = 2 if case["type"] == HALF else 4
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        # distinct words among t draws from frequencies 1 / rank
        z = math.log(v + 1.0)
        seen = sum(1.0 - (1.0 - math.log1p(1.0 / i) / z) ** t for i in range(1, v + 1))
        if case["op"] == "embedding":
            return {"bytes": int((seen + t + case["length"]) * d * size + 4 * t), "flops": 2 * t * d}
        return {"bytes": int((t + v) * d * size + 4 * t), "flops": t * d}
    size = 2 if case["type"] == HALF else 4
    n = sum(math.prod(x) for x in _model_shapes(case))
    return {"bytes": 2 * n * size, "flops": 3 * n}
