"""Measured cases of the row operators around a language model's matrix products: layer normalisation, embedding
lookup and distillation from a teacher's top logits, each with its gradient.

Every case names its operator (``op``: the public function), element type and sizes.  ``prepare`` makes the inputs on
the GPU from the seed, ``run`` is one pass -- elementary torch operations in 32 bits (64 for float64 data), or, with
``own`` set, the calls a user of ``dpnp_b200`` makes -- ``exact`` is the definition in 64 bits.
"""

import math

import torch

own = False

_TYPES = {"float16": torch.float16, "float32": torch.float32, "float64": torch.float64}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    """Training and serving passes of a model with a few thousand features and a vocabulary of 32 to 150 thousand."""
    return [
        # one token of a decoding step: nothing but latency
        dict(name="norm one token f16", op="layer_norm", dtype="float16", wtype="float16", rows=1, n=4096, pad=0),
        # the forward pass of a training batch, weights kept in 32 bits
        dict(name="norm batch f16", op="layer_norm", dtype="float16", wtype="float32", rows=16384, n=8192, pad=0),
        # a ragged batch, an odd width, rows that are a slice of wider ones
        dict(name="norm odd rows f32", op="layer_norm", dtype="float32", wtype="float32", rows=3001, n=1537, pad=6),
        # the backward pass of a training batch
        dict(name="norm gradient f16", op="layer_norm_backward", dtype="float16", wtype="float32", rows=16384, n=4096, pad=0),
        # the same for a small, odd width in 32 bits
        dict(name="norm gradient odd f32", op="layer_norm_backward", dtype="float32", wtype="float32", rows=5003, n=1023, pad=0),
        # the newest token of each of 8 sequences
        dict(name="embed one token f16", op="embedding", dtype="float16", tokens=8, vocab=32000, n=4096, scale=64.0),
        # a training batch's tokens
        dict(name="embed batch f16", op="embedding", dtype="float16", tokens=32768, vocab=128000, n=4096, scale=64.0),
        # gradient of a small table in 32 bits, odd vocabulary
        dict(name="embed gradient f32", op="embedding_backward", dtype="float32", tokens=8192, vocab=50257, n=768, scale=1.0),
        # gradient of a large table from a long batch
        dict(name="embed gradient f16", op="embedding_backward", dtype="float16", tokens=65536, vocab=128000, n=4096, scale=64.0),
        # the loss alone over a few rows (evaluation of a short answer), odd vocabulary
        dict(name="distil few rows f32", op="distillation_loss", dtype="float32", rows=7, vocab=50257, k=32, temperature=2.0),
        # loss and gradient of a training batch
        dict(name="distil step f16", op="distillation_loss_and_grad", dtype="float16", rows=4096, vocab=128000, k=64, temperature=1.0),
        # the gradient from kept statistics, odd vocabulary (rows start anywhere on the 16-byte grid)
        dict(name="distil gradient f32", op="distillation_loss_backward", dtype="float32", rows=1024, vocab=150001, k=100, temperature=1.5),
    ]


def _size(rng, low, high):
    """A size spread over the logarithm of low..high, odd half of the time."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:
        n |= 1
    return max(low, min(high, n))


def draw(rng):
    """One more case: the same operators from one row to long batches, narrow and wide, aligned and not."""
    op = rng.choice(["layer_norm", "layer_norm_backward", "embedding", "embedding_backward", "distillation_loss",
                     "distillation_loss_backward", "distillation_loss_and_grad"])
    dtype = rng.choice(["float16", "float16", "float16", "float32", "float32", "float64"])
    if op.startswith("layer_norm"):
        n = _size(rng, 33, 20000)
        rows = _size(rng, 1, max(1, min(30000, (1 << 26) // n)))
        wtype = rng.choice(["float16", "float32"]) if dtype == "float16" else dtype
        return dict(op=op, dtype=dtype, wtype=wtype, rows=rows, n=n, pad=rng.choice([0, 0, 1, 8]))
    if op.startswith("embedding"):
        n = _size(rng, 32, 8192)
        vocab = _size(rng, 500, max(500, min(150000, (1 << 27) // n)))
        tokens = _size(rng, 1, max(1, min(65536, (1 << 27) // n)))
        return dict(op=op, dtype=dtype, tokens=tokens, vocab=vocab, n=n, scale=rng.choice([1.0, math.sqrt(n)]))
    vocab = _size(rng, 1000, 150001)
    rows = _size(rng, 1, max(1, min(8192, (1 << 27) // vocab)))
    return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, k=_size(rng, 1, 128), temperature=rng.choice([1.0, 2.0, 0.7]))


_EPS = 1e-5


def _wide(dtype):
    return torch.float64 if dtype == torch.float64 else torch.float32


def prepare(case, seed):
    """The tensors a training or serving program holds before the call, made from the seed alone, and the buffers it
    keeps for the results; with ``own``, the library's arrays over the same memory as well."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    acc = _wide(dtype)

    def randn(*shape, of=acc):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(of)

    def empty(*shape, of=dtype):
        return torch.empty(*shape, device="cuda", dtype=of)

    s = {"case": case}
    if case["op"].startswith("layer_norm"):
        rows, n, wtype = case["rows"], case["n"], _TYPES[case["wtype"]]
        # activations with a spread and an offset of their own in every row; `pad` further columns behind each row
        spread, offset = randn(rows, 1).exp(), randn(rows, 1)
        s["x"] = (randn(rows, n + case["pad"]) * spread + offset).to(dtype)[:, :n]
        s["w"] = (1 + 0.1 * randn(n)).to(wtype)
        if case["op"] == "layer_norm":
            s["b"] = (0.1 * randn(n)).to(wtype)
            s["out"] = [empty(rows, n), empty(rows, of=acc), empty(rows, of=acc)]
        else:
            s["dy"] = randn(rows, n).to(dtype)
            wide = s["x"].double()
            mean = wide.mean(1)
            s["mean"] = mean.to(acc)
            s["rstd"] = ((wide - mean[:, None]).square().mean(1) + _EPS).rsqrt().to(acc)
            s["out"] = [empty(rows, n), empty(n, of=wtype), empty(n, of=wtype)]
    elif case["op"].startswith("embedding"):
        tokens, vocab, n = case["tokens"], case["vocab"], case["n"]
        # word frequencies fall as 1/rank, ranks are scattered over the vocabulary, and a few places are padding
        rank = (torch.rand(tokens, generator=gen, device="cuda", dtype=torch.float64) * math.log(vocab)).exp().long() - 1
        ids = (rank.clamp(0, vocab - 1) * 7919 + 13) % vocab
        ids[torch.rand(tokens, generator=gen, device="cuda") < 0.02] = -1
        s["ids"] = ids
        if case["op"] == "embedding":
            s["table"] = (0.02 * randn(vocab, n)).to(dtype)
            s["out"] = [empty(tokens, n)]
        else:
            s["dy"] = (0.01 * randn(tokens, n)).to(dtype)
            s["out"] = [empty(vocab, n)]
    else:
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        z = randn(rows, vocab, of=torch.float32).mul_(2.5).to(dtype)
        z[:, vocab - 5:] = torch.finfo(dtype).min                   # columns that fill the vocabulary up
        # k different words a row and the teacher's logits for them in falling order; short rows end in -1, and
        # a few rows (prompt, padding) have no teacher at all
        start = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
        step = torch.randint(1, max(2, (vocab - 5) // k), (rows, 1), generator=gen, device="cuda")
        index = (start + step * torch.arange(k, device="cuda")) % (vocab - 5)
        kept = torch.randint(1, 2 * k + 1, (rows, 1), generator=gen, device="cuda")
        index[torch.arange(k, device="cuda") >= kept] = -1
        index[rows - _unused(case):] = -1
        s["z"], s["index"] = z, index.int()
        s["t"] = (3 * randn(rows, k)).sort(dim=1, descending=True).values.to(acc)
        # the mean over the rows; 16-bit training scales its loss so that the gradients stay in that type's range
        s["g"] = torch.full((rows,), (65536.0 if dtype == torch.float16 else 1.0) / rows, device="cuda", dtype=acc)
        if case["op"] == "distillation_loss":
            s["out"] = [empty(rows, of=acc), empty(rows, 2, of=acc)]
        elif case["op"] == "distillation_loss_backward":
            top = z.amax(1).to(acc)
            total = torch.empty_like(top)
            for r in range(0, rows, 256):
                total[r:r + 256] = ((z[r:r + 256].double() - top[r:r + 256, None]) / case["temperature"]).exp().sum(1).log()
            used = (s["index"] >= 0).any(1)
            s["stats"] = torch.stack([torch.where(used, top, 0.0), torch.where(used, total, 0.0)], 1)
            s["out"] = [empty(rows, vocab)]
        else:
            s["out"] = [empty(rows, of=acc), empty(rows, vocab)]
    if own:
        import dpnp_b200 as dp

        # the arrays work on the stream that made the tensors
        queue = dp.StreamQueue(torch.cuda.current_device(), stream=torch.cuda.current_stream().cuda_stream)
        torch.cuda.current_stream().synchronize()
        view = lambda t: dp.from_dlpack(t, device=queue)  # noqa: E731
        s["arrays"] = {k: [view(t) for t in v] if k == "out" else view(v) for k, v in s.items()
                       if k == "out" or isinstance(v, torch.Tensor)}
    return s


def _unused(case):
    """Rows of a distillation case without a teacher."""
    return case["rows"] // 16


# -------------------------------------------------------------------------------------------------------------- runs
def run(state):
    case = state["case"]
    if own:
        return _own(state["arrays"], case, state["out"])
    return _PLAIN[case["op"]](state, case)


def _own(a, case, out):
    import dpnp_b200 as dp

    op = case["op"]
    if op == "layer_norm":
        dp.layer_norm(a["x"], a["w"], a["b"], eps=_EPS, return_stats=True, out=tuple(a["out"]))
    elif op == "layer_norm_backward":
        dp.layer_norm_backward(a["dy"], a["x"], a["mean"], a["rstd"], a["w"], out=tuple(a["out"]))
    elif op == "embedding":
        dp.embedding(a["table"], a["ids"], scale=case["scale"], out=a["out"][0])
    elif op == "embedding_backward":
        dp.embedding_backward(a["dy"], a["ids"], case["vocab"], scale=case["scale"], out=a["out"][0])
    elif op == "distillation_loss":
        dp.distillation_loss(a["z"], a["t"], a["index"], temperature=case["temperature"], return_stats=True,
                             out=tuple(a["out"]))
    elif op == "distillation_loss_backward":
        dp.distillation_loss_backward(a["g"], a["z"], a["t"], a["index"], a["stats"], temperature=case["temperature"],
                                      out=a["out"][0])
    else:
        dp.distillation_loss_and_grad(a["z"], a["t"], a["index"], a["g"], temperature=case["temperature"],
                                      out=tuple(a["out"]))
    return out


def _norm(s, case):
    x = s["x"].to(_wide(s["x"].dtype))
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1 / (d.square().mean(1, keepdim=True) + _EPS).sqrt()
    y = d * rstd * s["w"].to(x.dtype) + s["b"].to(x.dtype)
    return [y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]]


def _norm_gradient(s, case):
    acc = _wide(s["x"].dtype)
    x, dy, r = s["x"].to(acc), s["dy"].to(acc), s["rstd"][:, None]
    h = (x - s["mean"][:, None]) * r
    a = dy * s["w"].to(acc)
    dx = r * (a - a.mean(1, keepdim=True) - h * (a * h).mean(1, keepdim=True))
    return [dx.to(s["x"].dtype), (dy * h).sum(0).to(s["w"].dtype), dy.sum(0).to(s["w"].dtype)]


def _embed(s, case):
    ids = s["ids"]
    known = (ids >= 0) & (ids < case["vocab"])
    rows = s["table"][torch.where(known, ids, 0)].to(_wide(s["table"].dtype)) * case["scale"]
    return [torch.where(known[:, None], rows, 0.0).to(s["table"].dtype)]


def _embed_gradient(s, case):
    ids, vocab, acc = s["ids"], case["vocab"], _wide(s["dy"].dtype)
    known = (ids >= 0) & (ids < vocab)
    total = torch.zeros(vocab + 1, case["n"], device="cuda", dtype=acc)     # the last row takes the padding
    total.index_add_(0, torch.where(known, ids, vocab), s["dy"].to(acc))
    return [(total[:vocab] * case["scale"]).to(s["dy"].dtype)]


def _teacher(s, case, acc):
    """The teacher's distribution over its valid entries, and which entries and rows are valid."""
    t = s["t"].to(acc)
    valid = (s["index"] >= 0) & (s["index"] < case["vocab"]) & (t > -math.inf)
    t = torch.where(valid, t, -math.inf)
    top = t.amax(1, keepdim=True)
    e = torch.where(valid, ((t - top) / case["temperature"]).exp(), 0.0)
    total = e.sum(1, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    logp = torch.where(valid, (t - top) / case["temperature"] - total.log(), 0.0)
    return p, logp, valid, valid.any(1)


def _loss(s, case):
    acc, temp = _wide(s["z"].dtype), case["temperature"]
    z = s["z"].to(acc)
    p, logp, valid, used = _teacher(s, case, acc)
    top = z.amax(1)
    log_total = ((z - top[:, None]) / temp).exp().sum(1).log()
    at = z.gather(1, torch.where(valid, s["index"], 0).long())
    logq = (at - top[:, None]) / temp - log_total[:, None]
    loss = temp * temp * torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    zero = torch.zeros_like(loss)
    return torch.where(used, loss, zero), torch.stack([torch.where(used, top, zero), torch.where(used, log_total, zero)], 1)


def _distil_loss(s, case):
    return list(_loss(s, case))


def _gradient(s, case, stats):
    acc, temp = _wide(s["z"].dtype), case["temperature"]
    p, _, valid, used = _teacher(s, case, acc)
    dz = ((s["z"].to(acc) - stats[:, :1]) / temp - stats[:, 1:]).exp()
    dz.scatter_add_(1, torch.where(valid, s["index"], 0).long(), -p)
    dz = torch.where(used[:, None], dz * (s["g"][:, None] * temp), 0.0)
    return dz.to(s["z"].dtype)


def _distil_gradient(s, case):
    return [_gradient(s, case, s["stats"])]


def _distil_step(s, case):
    loss, stats = _loss(s, case)
    return [loss, _gradient(s, case, stats)]


_PLAIN = {
    "layer_norm": _norm, "layer_norm_backward": _norm_gradient, "embedding": _embed,
    "embedding_backward": _embed_gradient, "distillation_loss": _distil_loss,
    "distillation_loss_backward": _distil_gradient, "distillation_loss_and_grad": _distil_step,
}


# -------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Bytes that have to cross the memory once, and the arithmetic of the formulas."""
    s = {"float16": 2, "float32": 4, "float64": 8}
    es = s[case["dtype"]]
    acc = max(4, es)
    if case["op"].startswith("layer_norm"):
        rows, n, ws = case["rows"], case["n"], s[case["wtype"]]
        if case["op"] == "layer_norm":
            return {"bytes": 2 * rows * n * es + 2 * n * ws + 2 * rows * acc, "flops": 8 * rows * n}
        return {"bytes": 3 * rows * n * es + 3 * n * ws + 2 * rows * acc, "flops": 14 * rows * n}
    if case["op"].startswith("embedding"):
        tokens, vocab, n = case["tokens"], case["vocab"], case["n"]
        if case["op"] == "embedding":
            # distinct words among the tokens when a word of rank r has probability log(1 + 1/r) / log(vocab)
            seen, r = 0.0, 1
            while r < vocab:
                step = max(1, r // 16)
                seen += step * -math.expm1(-tokens * math.log1p(1 / (r + step / 2)) / math.log(vocab))
                r += step
            return {"bytes": (min(seen, tokens) + tokens) * n * es + 8 * tokens, "flops": tokens * n}
        return {"bytes": (tokens + vocab) * n * es + 8 * tokens, "flops": tokens * n}
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    used = rows - _unused(case)
    small = rows * k * (4 + acc) + 3 * rows * acc
    if case["op"] == "distillation_loss":
        return {"bytes": used * vocab * es + small, "flops": 4 * used * vocab}
    return {"bytes": (used + rows) * vocab * es + small, "flops": 8 * used * vocab}


# ------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """What ``run`` returns for these inputs, by the definitions in 64 bits."""
    s = prepare(case, seed)
    f = torch.float64
    op = case["op"]
    if op == "layer_norm":
        x = s["x"].to(f)
        mean = x.sum(1) / case["n"]
        var = torch.var(x, dim=1, correction=0)
        normal = torch.addcmul(s["b"].to(f), (x - mean[:, None]) / torch.sqrt(var + _EPS)[:, None], s["w"].to(f))
        return [normal, mean, torch.rsqrt(var + _EPS)]
    if op == "layer_norm_backward":
        # dx = J^T (dy w), with the Jacobian r (I - 1 1^T / n - h h^T / n) of the normalisation
        x, dy, n = s["x"].to(f), s["dy"].to(f), case["n"]
        h = (x - s["mean"].to(f)[:, None]).mul_(s["rstd"].to(f)[:, None])
        dw, db = torch.einsum("rn,rn->n", dy, h), dy.sum(0)
        a = dy.mul_(s["w"].to(f))
        proj = torch.einsum("rn,rn->r", a, h) / n
        dx = (a - (a.sum(1) / n)[:, None] - h.mul_(proj[:, None])).mul_(s["rstd"].to(f)[:, None])
        return [dx, dw, db]
    if op == "embedding":
        table = torch.cat([s["table"].to(f) * case["scale"], torch.zeros(1, case["n"], device="cuda", dtype=f)])
        return [table[s["ids"]]]                                             # -1 is the row of zeros at the end
    if op == "embedding_backward":
        keep = s["ids"] >= 0
        ids, dy = s["ids"][keep], s["dy"][keep].to(f)
        out = torch.zeros(case["vocab"], case["n"], device="cuda", dtype=f)
        return [out.scatter_add_(0, ids[:, None].expand_as(dy), dy).mul_(case["scale"])]
    temp, index = case["temperature"], s["index"].long()
    here = index >= 0
    used = here.any(1)
    p = torch.softmax(torch.where(here, s["t"].to(f) / temp, -math.inf), 1).nan_to_num(0.0)
    rows, loss, stats, grads = case["rows"], [], [], []
    for r in range(0, rows, 512):
        z, at, w = s["z"][r:r + 512].to(f) / temp, index[r:r + 512].clamp(min=0), p[r:r + 512]
        u = used[r:r + 512]
        lse = torch.logsumexp(z, 1)
        kl = (torch.xlogy(w, w) - w * (z.gather(1, at) - lse[:, None])).sum(1)
        loss.append(torch.where(u, kl * temp**2, 0.0))
        top = z.amax(1)
        stats.append(torch.stack([torch.where(u, top * temp, 0.0), torch.where(u, lse - top, 0.0)], 1))
        if op != "distillation_loss":
            if op == "distillation_loss_backward":                           # the statistics are inputs there
                lse = s["stats"][r:r + 512, 0].to(f) / temp + s["stats"][r:r + 512, 1].to(f)
            q = torch.exp(z - lse[:, None])
            q.scatter_add_(1, at, -w)
            grads.append(q.mul_(s["g"][r:r + 512, None].to(f) * temp * u[:, None]))
    if op == "distillation_loss":
        return [torch.cat(loss), torch.cat(stats)]
    if op == "distillation_loss_backward":
        return [torch.cat(grads)]
    return [torch.cat(loss), torch.cat(grads)]
