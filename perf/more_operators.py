"""Performance cases of the operators that training on packed documents adds: attention under document and prefix masks with a
score cap and a distance bias, layer norm, the scaled embedding with its table's gradient, and clipping by the global norm.

`listed()` names the cases, `draw(rng)` makes another one of the same ranges, `prepare` builds what a program has in hand
before the call, `run` makes one pass: with `own` through the package's entry points, without it in elementary torch
operations (float32 whatever the inputs' type, rounded once at the end), `exact` is the same from the definitions in float64,
`work` the traffic and arithmetic that no implementation can avoid.

Sizes are those of the model configuration (14 query heads over 2 key heads of 64, hidden size 896, 24 layers, vocabulary 151936)
and of the tests (hidden 777 and 1000, vocabularies 32000 and 50257); sequences go from a few tokens to 16384.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # a training pass over packed documents (some 600 tokens each) and a little padding, the model's own heads
        dict(name="attention_packed", kind="attention", train=True, batch=2, seq=4096, kv_heads=2, groups=7, dim=64, dtype="bf16",
             documents=7, padding=0.03, prefix=0.0, softcap=0.0, bias=False, token_major=True),
        # scoring one long text whose prompt is read in both directions: forward only
        dict(name="attention_prefix_long", kind="attention", train=False, batch=1, seq=16384, kv_heads=2, groups=7, dim=64, dtype="bf16",
             documents=2, padding=0.0, prefix=0.4, softcap=0.0, bias=False, token_major=True),
        # a training pass with capped scores, whole causal sequences, two query heads to a key head
        dict(name="attention_capped", kind="attention", train=True, batch=4, seq=1024, kv_heads=8, groups=2, dim=64, dtype="bf16",
             documents=1, padding=0.0, prefix=0.0, softcap=30.0, bias=False, token_major=False),
        # a training pass with a distance bias, one key head to a query head, odd length
        dict(name="attention_bias_odd", kind="attention", train=True, batch=3, seq=777, kv_heads=12, groups=1, dim=64, dtype="bf16",
             documents=3, padding=0.1, prefix=0.0, softcap=0.0, bias=True, token_major=True),
        # a few tokens in float32, everything on: a validation run, latency
        dict(name="attention_small_f32", kind="attention", train=True, batch=1, seq=19, kv_heads=2, groups=3, dim=64, dtype="f32",
             documents=3, padding=0.1, prefix=0.3, softcap=20.0, bias=True, token_major=False),
        # one decoding batch's worth of rows in float32
        dict(name="layer_norm_small", kind="layer_norm", rows=16, dim=896, dtype="f32", residual=False),
        # a training step's tokens, with the gradient of the residual path
        dict(name="layer_norm_32768", kind="layer_norm", rows=32768, dim=896, dtype="bf16", residual=True),
        # odd rows and columns
        dict(name="layer_norm_odd_f32", kind="layer_norm", rows=8191, dim=777, dtype="f32", residual=False),
        # a short text with a small table in float32: latency
        dict(name="embedding_small", kind="embedding", tokens=17, dim=128, vocab=1000, dtype="f32", padding=0.0, scale=1.0),
        # a training step's tokens over the full vocabulary, frequencies as in text, some padding
        dict(name="embedding_8192", kind="embedding", tokens=8192, dim=896, vocab=151936, dtype="bf16", padding=0.05, scale=29.933),
        # the gradients of rank 8 adapters on four projections of 24 layers
        dict(name="clip_adapters", kind="clip", tensors=192, numel=2500000, dtype="f32"),
        # the gradients of a whole model
        dict(name="clip_model", kind="clip", tensors=290, numel=250000001, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "layer_norm", "embedding", "clip"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind == "attention":
        train = rng.random() < 0.7
        groups, kv_heads = rng.choice([(7, 2), (1, 4), (1, 12), (2, 8), (4, 2), (3, 1), (7, 1)])
        seq = _log(rng, 2, 6000 if dtype == "bf16" else 1200)
        most = (4 * 10 ** 8 if dtype == "bf16" else 3 * 10 ** 7) // (seq * seq * groups * kv_heads)
        batch = max(1, min(8, most, _log(rng, 1, 8)))
        return dict(kind=kind, train=train, batch=batch, seq=seq, kv_heads=kv_heads, groups=groups,
                    dim=64 if dtype == "bf16" else rng.choice([64, 64, 32, 80, 128]), dtype=dtype,
                    documents=min(seq, _log(rng, 1, 24)), padding=rng.choice([0.0, 0.0, round(rng.uniform(0.0, 0.4), 2)]),
                    prefix=rng.choice([0.0, 0.0, round(rng.uniform(0.1, 1.0), 2)]), softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                    bias=rng.random() < 0.3, token_major=rng.random() < 0.5)
    if kind == "layer_norm":
        dim = rng.choice([896, 1024, 768, _log(rng, 16, 8192), _log(rng, 16, 8192) | 1])
        rows = _log(rng, 1, min(100000, 6 * 10 ** 7 // dim))
        return dict(kind=kind, rows=rows, dim=dim, dtype=dtype, residual=rng.random() < 0.4)
    if kind == "embedding":
        vocab = rng.choice([151936, 50257, 32000, _log(rng, 100, 160000)])
        dim = rng.choice([896, 768, _log(rng, 16, 4096), 8 * _log(rng, 2, 512)])
        dim = min(dim, 14 * 10 ** 7 // vocab)
        tokens = _log(rng, 1, min(65536, 6 * 10 ** 7 // dim))
        return dict(kind=kind, tokens=tokens, dim=dim, vocab=vocab, dtype=dtype, padding=rng.choice([0.0, round(rng.uniform(0.0, 0.5), 2)]),
                    scale=rng.choice([1.0, round(math.sqrt(dim), 3)]))
    numel = _log(rng, 1000, 2 * 10 ** 8)
    return dict(kind=kind, tensors=min(numel, _log(rng, 1, 600)), numel=numel, dtype=dtype)


def _parts(case, total, count, rng):
    """`total` cut into `count` parts of at least one, of sizes that differ as those of documents and parameters do."""
    weights = [math.exp(rng.gauss(0.0, 0.7)) for _ in range(count)]
    cut = (total - count) / sum(weights)
    sizes = [1 + int(w * cut) for w in weights]
    sizes[0] += total - sum(sizes)
    return sizes


def _documents(case):
    """Per sequence its documents as (length, length of the part that is read in both directions); the same for every seed."""
    rng = random.Random("%(batch)d %(seq)d %(documents)d %(padding).2f %(prefix).2f" % case)
    out = []
    for _ in range(case["batch"]):
        used = max(1, case["seq"] - int(case["seq"] * case["padding"] * rng.uniform(0.5, 1.0)))
        sizes = _parts(case, used, min(case["documents"], used), rng)
        out.append([(n, int(n * case["prefix"] * rng.uniform(0.5, 1.0))) for n in sizes])
    return out


def work(case):
    kind, size = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind == "attention":
        pairs = sum(n * (n + 1) // 2 + p * (p - 1) // 2 for docs in _documents(case) for n, p in docs)
        heads, rows = case["kv_heads"] * case["groups"], case["batch"] * case["seq"]
        q, kv, lse = rows * heads * case["dim"] * size, rows * case["kv_heads"] * case["dim"] * size, rows * heads * 4
        # q, k, v, o; the training pass also d o, and d q, d k, d v
        traffic = 2 * q + 2 * kv + lse + (2 * q + 2 * kv if case["train"] else 0)
        return {"bytes": traffic + rows * 5, "flops": pairs * heads * case["dim"] * (14 if case["train"] else 4)}
    if kind == "layer_norm":
        n = case["rows"] * case["dim"]
        return {"bytes": n * size * (4 + case["residual"]) + case["dim"] * (2 * size + 8), "flops": 16 * n}
    if kind == "embedding":
        n = case["tokens"] * case["dim"]
        return {"bytes": n * size * 3 + case["vocab"] * case["dim"] * 4 + case["tokens"] * 4, "flops": 2 * n}
    return {"bytes": 2 * case["numel"] * size, "flops": 3 * case["numel"]}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, device=dev, generator=gen)  # noqa: E731
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    state = dict(case=case)
    if kind == "attention":
        B, S, d, heads = case["batch"], case["seq"], case["dim"], case["kv_heads"] * case["groups"]
        nb, gs = B * case["kv_heads"], case["groups"] * S
        order = random.Random(seed)
        ids, prefix = torch.full((B, S), -1, dtype=torch.int32), torch.zeros(B, S, dtype=torch.bool)
        for b, docs in enumerate(_documents(case)):
            order.shuffle(docs)
            at = 0
            for i, (n, p) in enumerate(docs):
                ids[b, at:at + n] = i
                prefix[b, at:at + p] = True
                at += n
        state.update(ids=ids.to(dev), prefix=prefix.to(dev) if case["prefix"] > 0 else None)
        # scores of a trained head: a standard deviation of 2 or so, more where a cap has something to do
        state["q"] = (rand(nb, gs, d) * (6.0 if case["softcap"] > 0 else 2.0)).to(dt)
        state["k"], state["v"] = rand(nb, S, d).to(dt), rand(nb, S, d).to(dt)
        state["slopes"] = 2.0 ** (-8.0 * (torch.arange(heads, device=dev) + 1) / heads) if case["bias"] else None
        state["dout"] = (rand(B * S, heads * d) if case["token_major"] else rand(nb, gs, d)).to(dt) if case["train"] else None
        return state
    if kind == "layer_norm":
        M, D = case["rows"], case["dim"]
        # activations with a mean of their own in each row and a few wide columns
        x = rand(M, D) + 0.5 * rand(M, 1)
        x[:, :: max(1, D // 7)] *= 8.0
        state.update(x=x.to(dt), w=(1 + 0.2 * rand(D)).to(dt), b=(0.1 * rand(D)).to(dt), dy=rand(M, D).to(dt))
        state["residual"] = rand(M, D).to(dt) if case["residual"] else None
        return state
    if kind == "embedding":
        M, V = case["tokens"], case["vocab"]
        # token frequencies fall off as the rank's reciprocal, ranks scattered over the ids
        rank = torch.exp(torch.rand(M, device=dev, generator=gen) * math.log(V)).long().clamp_(1, V) - 1
        ids = torch.randperm(V, device=dev, generator=gen)[rank].to(torch.int32)
        ids = torch.where(torch.rand(M, device=dev, generator=gen) < case["padding"], torch.full_like(ids, -1), ids)
        state.update(ids=ids, table=(0.02 * rand(V, case["dim"])).to(dt), dout=rand(M, case["dim"]).to(dt))
        return state
    sizes = _parts(case, case["numel"], case["tensors"], random.Random(case["numel"]))
    grads = [t.clone() for t in (rand(case["numel"]) * 0.01).to(dt).split(sizes)]
    out = torch.empty(case["numel"], dtype=dt, device=dev)   # the clipped gradients, one behind the other
    state.update(grads=grads, out=out)
    if own:
        from metal_candle_b200 import training

        # gradient buffers stay where they are from step to step, and so does what knows them
        state["clipper"] = training.GradClipper(grads, out=list(out.split(sizes)))
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _visible(ids, prefix):
    """[B, S queries, S keys]: both in the same run of equal ids that are not negative, and the key no later than the query or in the
    run's leading stretch of prefix positions."""
    B, S = ids.shape
    at = torch.arange(S, device=ids.device).expand(B, S)
    first = torch.ones_like(ids, dtype=torch.bool)
    first[:, 1:] = ids[:, 1:] != ids[:, :-1]
    start = torch.where(first, at, torch.zeros_like(at)).cummax(1).values
    seen = at[:, None, :] <= at[:, :, None]
    if prefix is not None:
        broken = torch.where(prefix, torch.full_like(at, -1), at).cummax(1).values   # the last position that is no prefix
        seen = seen | (broken < start)[:, None, :]
    return (start[:, None, :] == start[:, :, None]) & seen & (ids >= 0)[:, :, None]


def _plain_attention(st):
    case = st["case"]
    B, S, Hk, G, d = case["batch"], case["seq"], case["kv_heads"], case["groups"], case["dim"]
    q = st["q"].float().view(B, Hk, G, S, d)
    k, v = st["k"].float().view(B, Hk, 1, S, d), st["v"].float().view(B, Hk, 1, S, d)
    scale, cap, dt = 1.0 / math.sqrt(d), case["softcap"], st["q"].dtype
    visible = _visible(st["ids"], st["prefix"])[:, None, None]
    s = (q @ k.transpose(-1, -2)).mul_(scale)
    bent = None
    if cap > 0:
        bent = (s / cap).tanh_()
        s = bent * cap
    if st["slopes"] is not None:
        at = torch.arange(S, device=q.device)
        s = s - st["slopes"].view(1, Hk, G, 1, 1) * (at[:, None] - at[None, :]).abs()
    s = s.masked_fill_(~visible, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - top.clamp_min(-3e38)).exp_()
    del s
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.clamp_min(1e-38))
    o = p @ v
    lse = (top + total.log()).view(B * Hk, G * S)
    major = (lambda t: t.permute(0, 3, 1, 2, 4).reshape(B * S, Hk * G * d)) if case["token_major"] else (lambda t: t.reshape(B * Hk, G * S, d))  # noqa: E731
    if not case["train"]:
        return major(o).to(dt), lse
    do = st["dout"].float()
    do = do.view(B, S, Hk, G, d).permute(0, 2, 3, 1, 4) if case["token_major"] else do.view(B, Hk, G, S, d)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = (do @ v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if cap > 0:
        ds = ds * (1 - bent * bent)
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2) * scale
    return (major(o).to(dt), lse, dq.view(B * Hk, G * S, d).to(dt), dk.reshape(B * Hk, S, d).to(dt), dv.reshape(B * Hk, S, d).to(dt))


def _run_plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "attention":
        return _plain_attention(st)
    if kind == "layer_norm":
        x, w, dy = st["x"].float(), st["w"].float(), st["dy"].float()
        off = x - x.mean(-1, keepdim=True)
        rstd = ((off * off).mean(-1, keepdim=True) + EPS).rsqrt()
        n = off * rstd
        y = n * w + st["b"].float()
        g = dy * w
        dx = (g - g.mean(-1, keepdim=True) - n * (g * n).mean(-1, keepdim=True)) * rstd
        if st["residual"] is not None:
            dx = dx + st["residual"].float()
        return y.to(st["x"].dtype), dx.to(st["x"].dtype), (dy * n).sum(0), dy.sum(0)
    if kind == "embedding":
        ids, table, dout = st["ids"], st["table"], st["dout"].float()
        kept = (ids >= 0) & (ids < case["vocab"])
        at = torch.where(kept, ids, torch.zeros_like(ids)).long()
        out = torch.where(kept[:, None], table[at].float() * case["scale"], torch.zeros((), device=ids.device)).to(table.dtype)
        grad = torch.zeros(case["vocab"], case["dim"], device=ids.device)
        grad.index_add_(0, at, torch.where(kept[:, None], dout * case["scale"], torch.zeros((), device=ids.device)))
        return out, grad
    g = torch.cat(st["grads"]).float()
    norm = g.double().square().sum().sqrt().float().view(1)
    st["out"].copy_(g * (1.0 / (norm + 1e-6)).clamp_max(1.0))
    return norm, st["out"]


# ---- the framework's operators --------------------------------------------------------------------------------------------

def _run_own(st):
    from metal_candle_b200 import backend

    case = st["case"]
    kind = case["kind"]
    if kind == "attention":
        q, k, v = st["q"], st["k"], st["v"]
        how = dict(groups=case["groups"], scale=1.0 / math.sqrt(case["dim"]), softcap=case["softcap"], slopes=st["slopes"],
                   token_major=case["token_major"], mask=backend.attention_mask(st["ids"], st["prefix"]))
        o, lse = backend.attention_masked_forward(q, k, v, **how)
        if not case["train"]:
            return o, lse
        return (o, lse, *backend.attention_masked_backward(q, k, v, o, lse, st["dout"], **how))
    if kind == "layer_norm":
        y = backend.layer_norm_fused(st["x"], st["w"], st["b"], EPS)
        return (y, *backend.layer_norm_backward(st["x"], st["w"], st["dy"], EPS, dx_residual=st["residual"]))
    if kind == "embedding":
        out = backend.embedding(st["ids"], st["table"], scale=case["scale"])
        return out, backend.embedding_backward(st["ids"], st["dout"], case["vocab"], scale=case["scale"])
    return st["clipper"].clip(1.0), st["out"]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in float64 --------------------------------------------------------------------------------------------

def _exact_attention(case, st):
    B, S, Hk, G, d = case["batch"], case["seq"], case["kv_heads"], case["groups"], case["dim"]
    dev, f64 = st["q"].device, torch.float64
    q, k, v = (t.double() for t in (st["q"].view(B, Hk, G, S, d), st["k"].view(B, Hk, S, d), st["v"].view(B, Hk, S, d)))
    do = None
    if case["train"]:
        do = st["dout"].double()
        do = do.view(B, S, Hk, G, d).permute(0, 2, 3, 1, 4) if case["token_major"] else do.view(B, Hk, G, S, d)
    o, dq = torch.zeros(B, Hk, G, S, d, dtype=f64, device=dev), torch.zeros(B, Hk, G, S, d, dtype=f64, device=dev)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    lse = torch.full((B, Hk, G, S), -math.inf, dtype=f64, device=dev)
    ids, prefix = st["ids"].tolist(), None if st["prefix"] is None else st["prefix"].tolist()
    for b in range(B):
        at = 0
        while at < S:
            end = at + 1
            while end < S and ids[b][end] == ids[b][at]:
                end += 1
            if ids[b][at] >= 0:
                n, lead = end - at, 0
                while prefix is not None and lead < n and prefix[b][at + lead]:
                    lead += 1
                pos = torch.arange(n, device=dev)
                hidden = (pos[None, :] > pos[:, None]) & (pos[None, :] >= lead)
                cut = slice(at, end)
                for h in range(Hk):
                    for g in range(G):
                        a, c, e = (t.detach().requires_grad_(case["train"]) for t in (q[b, h, g, cut], k[b, h, cut], v[b, h, cut]))
                        s = a @ c.T / math.sqrt(d)
                        if case["softcap"] > 0:
                            s = case["softcap"] * torch.tanh(s / case["softcap"])
                        if st["slopes"] is not None:
                            s = s - st["slopes"][h * G + g].double() * (pos[:, None] - pos[None, :]).abs()
                        s = s.masked_fill(hidden, -math.inf)
                        z = torch.logsumexp(s, -1)
                        r = torch.exp(s - z[:, None]) @ e
                        o[b, h, g, cut], lse[b, h, g, cut] = r.detach(), z.detach()
                        if case["train"]:
                            ga, gc, ge = torch.autograd.grad(r, (a, c, e), do[b, h, g, cut])
                            dq[b, h, g, cut] = ga
                            dk[b, h, cut] += gc
                            dv[b, h, cut] += ge
            at = end
    o = o.permute(0, 3, 1, 2, 4).reshape(B * S, Hk * G * d) if case["token_major"] else o.view(B * Hk, G * S, d)
    if not case["train"]:
        return o, lse.view(B * Hk, G * S)
    return o, lse.view(B * Hk, G * S), dq.view(B * Hk, G * S, d), dk.view(B * Hk, S, d), dv.view(B * Hk, S, d)


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind == "attention":
        return _exact_attention(case, st)
    if kind == "layer_norm":
        x, w, b = (st[n].double().requires_grad_(True) for n in ("x", "w", "b"))
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * w + b
        dx, dw, db = torch.autograd.grad(y, (x, w, b), st["dy"].double())
        return y.detach(), dx if st["residual"] is None else dx + st["residual"].double(), dw, db
    if kind == "embedding":
        V, scale = case["vocab"], float(torch.tensor(case["scale"], dtype=torch.float32))
        table = torch.cat([st["table"].double(), torch.zeros(1, case["dim"], dtype=torch.float64, device=st["table"].device)])
        at = torch.where((st["ids"] >= 0) & (st["ids"] < V), st["ids"].long(), torch.full_like(st["ids"], V).long())
        grad = torch.zeros_like(table).index_put_((at,), st["dout"].double() * scale, accumulate=True)
        return table[at] * scale, grad[:V]
    flat = torch.cat(st["grads"]).double()
    norm = torch.linalg.vector_norm(flat)
    return norm.view(1), flat * min(1.0, 1.0 / (float(norm) + 1e-6))
