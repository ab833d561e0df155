"""Performance cases of the operators that post-training adds to the training step: losses over the logits of given tokens.

`listed()` names the cases, `draw(rng)` makes another one of the same ranges, `prepare` builds what a program has in hand
before the call, `run` makes one pass: with `own` through the package's entry points, without it in elementary torch
operations (float32 whatever the logits' type, rounded once at the end), `exact` is the same from the definitions in float64,
`work` the traffic and arithmetic that no implementation can avoid.

Vocabularies are those of the model configuration (151936) and of the tests (32000, 50257); token counts go from one token
to a batch of 4096.  Positions whose target is -100 (prompt and padding) are ignored.
"""
import math

import torch

own = False

IGNORE = -100
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # scoring one sampled token under a frozen policy: the smallest call, latency
        dict(name="score_one_token", kind="score", batch=1, seq=1, vocab=151936, dtype="bf16", temperature=1.0, keep=1.0),
        # the reference model's log-probabilities of a batch of answers, forward only
        dict(name="score_2048", kind="score", batch=4, seq=512, vocab=151936, dtype="bf16", temperature=1.0, keep=0.8),
        # log-probabilities with their reverse pass, for a loss of the user's own; odd vocabulary and length
        dict(name="logprob_odd", kind="logprob", batch=3, seq=333, vocab=50257, dtype="bf16", temperature=0.7, keep=0.7),
        # the same for one short text in float32
        dict(name="logprob_small", kind="logprob", batch=1, seq=16, vocab=32000, dtype="f32", temperature=1.0, keep=1.0),
        # one short preference pair in float32: a validation run
        dict(name="preference_small", kind="preference", pairs=1, seq=19, vocab=1000, dtype="f32", smoothing=0.0, average=False, keep=0.6),
        # a batch of preference pairs over the full vocabulary, loss and gradient
        dict(name="preference_2048", kind="preference", pairs=4, seq=256, vocab=151936, dtype="bf16", smoothing=0.0, average=False, keep=0.6),
        # length-normalised pairs with smoothed labels, float32, odd length
        dict(name="preference_f32", kind="preference", pairs=3, seq=127, vocab=32000, dtype="f32", smoothing=0.1, average=True, keep=0.8),
        # a policy update on one short answer
        dict(name="policy_small", kind="policy", batch=1, seq=8, vocab=151936, dtype="bf16", temperature=1.0, keep=1.0, kl=0.04,
             sequence_mean=False, per_token=False),
        # a policy update on eight answers of a group, with the KL term
        dict(name="policy_4096", kind="policy", batch=8, seq=512, vocab=151936, dtype="bf16", temperature=1.0, keep=0.75, kl=0.04,
             sequence_mean=True, per_token=False),
        # advantages for each token, a sampling temperature, no KL term, odd vocabulary and length; float32 logits
        dict(name="policy_odd_f32", kind="policy", batch=5, seq=101, vocab=50257, dtype="f32", temperature=0.7, keep=0.9, kl=0.0,
             sequence_mean=False, per_token=True),
        # distillation of a batch from 64 teacher entries a token at temperature 2
        dict(name="distill_2048", kind="distill", batch=2, seq=1024, vocab=151936, top=64, dtype="bf16", temperature=2.0, keep=0.9),
        # odd sizes throughout, float32
        dict(name="distill_odd_f32", kind="distill", batch=3, seq=67, vocab=50257, top=101, dtype="f32", temperature=1.5, keep=0.8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["score", "logprob", "preference", "policy", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    vocab = rng.choice([151936, 50257, 32000, _log(rng, 1000, 160000), _log(rng, 1000, 160000) | 1])
    most = (5 * 10 ** 8 if dtype == "bf16" else 2 * 10 ** 8) // vocab
    tokens = _log(rng, 2, min(most, 20000))
    batch = max(2 if kind == "preference" else 1, min(tokens // 2, _log(rng, 1, 16)))
    seq = max(1, tokens // batch)
    keep = rng.choice([1.0, round(rng.uniform(0.3, 1.0), 2)])
    temperature = rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)])
    case = dict(kind=kind, vocab=vocab, dtype=dtype, seq=seq, keep=keep)
    if kind == "preference":
        case.update(pairs=batch // 2, smoothing=rng.choice([0.0, 0.1]), average=rng.random() < 0.3)
        return case
    case.update(batch=batch, temperature=temperature)
    if kind == "policy":
        case.update(kl=rng.choice([0.0, 0.04, 0.2]), sequence_mean=rng.random() < 0.5, per_token=rng.random() < 0.5)
    if kind == "distill":
        case.update(top=_log(rng, 1, 256))
    return case


def _rows(case):
    return 2 * case["pairs"] if case["kind"] == "preference" else case["batch"]


def work(case):
    M, V = _rows(case) * case["seq"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    sweeps = 1 if case["kind"] == "score" else 2
    extra = {"score": 16, "logprob": 20, "preference": 12, "policy": 28, "distill": 1 + 6 * case.get("top", 0)}[case["kind"]]
    kept = case["keep"]
    # an ignored position's logits need not be read; its gradient (zeros) has to be written
    return {"bytes": M * V * size * (kept + sweeps - 1) + M * extra, "flops": M * V * kept * (3 if sweeps == 1 else 5)}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _make_logits(case, rows, seq, gen, dev):
    """Logits as a language model has them: a broad bulk, and the token that was sampled near the top."""
    V, dt = case["vocab"], DTYPES[case["dtype"]]
    M = rows * seq
    logits = torch.empty(M, V, dtype=dt, device=dev)
    targets = torch.randint(0, V, (M,), device=dev, generator=gen)
    lift = torch.rand(M, device=dev, generator=gen) * 14
    step = max(1, (1 << 28) // V)
    for i in range(0, M, step):
        part = torch.randn(min(step, M - i), V, device=dev, generator=gen) * 2.5
        part[torch.arange(part.shape[0], device=dev), targets[i:i + step]] += lift[i:i + step]
        logits[i:i + step] = part.to(dt)
    kept = torch.rand(M, device=dev, generator=gen) < case["keep"]
    kept[0] = True
    return logits.view(rows, seq, V), targets, kept


def _log_probs(logits, targets, temperature):
    """float32 log-probabilities, some rows at a time."""
    x2, V = logits.view(-1, logits.shape[-1]), logits.shape[-1]
    out = torch.empty(x2.shape[0], device=logits.device)
    step = max(1, (1 << 28) // V)
    for i in range(0, x2.shape[0], step):
        y = x2[i:i + step].float() / temperature
        top = y.amax(-1, keepdim=True)
        lse = top[:, 0] + (y - top).exp().sum(-1).log()
        out[i:i + step] = y.gather(1, targets[i:i + step, None])[:, 0] - lse
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, seq, kind = _rows(case), case["seq"], case["kind"]
    logits, targets, kept = _make_logits(case, rows, seq, gen, dev)
    state = dict(case=case, logits=logits)
    masked = torch.where(kept, targets, torch.full_like(targets, IGNORE)).view(rows, seq)
    rand = lambda *shape: torch.randn(*shape, device=dev, generator=gen)  # noqa: E731
    if kind == "distill":
        K, M = case["top"], rows * seq
        # the teacher's largest logits: some of the student's own candidates (the target first), others anywhere, no id twice
        first = targets[:, None]
        stride = torch.randint(1, max(2, (case["vocab"] - 1) // K), (M, 1), device=dev, generator=gen)
        state["teacher_ids"] = ((first + stride * torch.arange(K, device=dev)) % case["vocab"]).view(rows, seq, K)
        best = 6 + 3 * rand(M, 1)
        state["teacher_logits"] = (best - 5 * torch.rand(M, K, device=dev, generator=gen).cumsum(1) / (1 + K / 8)).to(
            DTYPES[case["dtype"]]).view(rows, seq, K)
        state["mask"] = kept.view(rows, seq)
        return state
    state["targets"] = masked
    if kind == "logprob":
        state["dlogp"] = rand(rows, seq) / (rows * seq)
    elif kind == "preference":
        logp = torch.where(kept, _log_probs(logits, targets, 1.0), torch.zeros((), device=dev)).view(rows, seq).sum(-1)
        if case["average"]:
            logp = logp / kept.view(rows, seq).sum(-1).clamp_min(1)
        # the frozen reference a few nats away
        state["ref"] = logp + rand(rows) * (0.5 if case["average"] else 4.0)
    elif kind == "policy":
        logp = _log_probs(logits, targets, case["temperature"]).view(rows, seq)
        drift = rand(rows, seq) * 0.15
        # a ratio within rounding of a clipping border may fall on either side of it: such tokens are moved off
        for border in (0.8, 1.2):
            drift = torch.where((drift.exp() - border).abs() < 2e-3, drift + 8e-3, drift)
        state["old"] = logp - drift
        state["ref"] = logp + rand(rows, seq) * 0.3 if case["kl"] > 0 else None
        state["advantages"] = rand(rows, seq) if case["per_token"] else rand(rows)
    return state


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _softmax_parts(logits, temperature):
    """y = x / T, its log-sum-exp and probabilities, in float32."""
    y = logits.float()
    if temperature != 1.0:
        y = y / temperature
    top = y.amax(-1, keepdim=True)
    e = (y - top).exp()
    s = e.sum(-1, keepdim=True)
    return y, top + s.log(), e / s


def _row_gradient(p, targets, kept, coef, dtype):
    """coef * (onehot(target) - p) for kept rows, zeros for the others."""
    g = p * -coef[..., None]
    g.scatter_add_(-1, targets.clamp_min(0)[..., None], coef[..., None])
    g = torch.where(kept[..., None], g, torch.zeros((), device=g.device))
    return g.to(dtype)


def _plain_log_probs(logits, targets, temperature):
    y, lse, p = _softmax_parts(logits, temperature)
    kept = targets != IGNORE
    zero = torch.zeros((), device=y.device)
    logp = torch.where(kept, y.gather(-1, targets.clamp_min(0)[..., None])[..., 0] - lse[..., 0], zero)
    return logp, torch.where(kept, lse[..., 0], zero), p, kept


def _softplus(z):
    return z.clamp_min(0) + (1 + (-z.abs()).exp()).log()


def _run_plain(st):
    case, logits = st["case"], st["logits"]
    kind = case["kind"]
    if kind == "distill":
        T = case["temperature"]
        y, lse, p = _softmax_parts(logits, T)
        _, tlse, q = _softmax_parts(st["teacher_logits"], T)
        log_q = st["teacher_logits"].float() / T - tlse
        kept, n = st["mask"], st["mask"].sum().clamp_min(1)
        rows = (q * (log_q - (y.gather(-1, st["teacher_ids"]) - lse))).sum(-1) * (T * T)
        loss = (torch.where(kept, rows, torch.zeros((), device=y.device)).double().sum() / n).float().view(1)
        g = p.scatter_add_(-1, st["teacher_ids"], -q)
        g = torch.where(kept[..., None], g * (T / n), torch.zeros((), device=g.device))
        return loss, g.to(logits.dtype)
    targets = st["targets"]
    logp, lse, p, kept = _plain_log_probs(logits, targets, case.get("temperature", 1.0))
    if kind == "score":
        return logp, lse
    if kind == "logprob":
        return logp, _row_gradient(p, targets, kept, st["dlogp"] / case["temperature"], logits.dtype)
    if kind == "preference":
        pairs, eps, beta = case["pairs"], case["smoothing"], 0.1
        w = 1.0 / kept.sum(-1).clamp_min(1).float() if case["average"] else torch.ones(2 * pairs, device=logp.device)
        sums = (logp.double().sum(-1) * w).float()
        margin = sums - st["ref"]
        z = beta * (margin[:pairs] - margin[pairs:])
        loss = ((1 - eps) * _softplus(-z) + eps * _softplus(z)).mean().view(1)
        dz = (eps - 1 / (1 + z.exp())) * (beta / pairs)   # sigma(z) - (1 - eps)
        coef = torch.cat([dz, -dz]) * w
        return loss, sums, _row_gradient(p, targets, kept, coef[:, None].expand_as(logp), logits.dtype)
    A = st["advantages"] if case["per_token"] else st["advantages"][:, None].expand_as(logp)
    ratio = (logp - st["old"]).exp()
    clipped = ratio.clamp(0.8, 1.2)
    terms = -torch.minimum(ratio * A, clipped * A)
    passes = torch.where(A >= 0, ratio <= 1.2, ratio >= 0.8)
    dterm = torch.where(passes, -A * ratio, torch.zeros((), device=A.device))
    if case["kl"] > 0:
        d = st["ref"] - logp
        terms = terms + case["kl"] * (d.exp() - d - 1)
        dterm = dterm + case["kl"] * (1 - d.exp())
    count = kept.sum(-1, keepdim=True)
    if case["sequence_mean"]:
        weight = 1.0 / (count.clamp_min(1) * (count > 0).sum().clamp_min(1)).float()
    else:
        weight = 1.0 / count.sum().clamp_min(1).float().view(1, 1)
    zero = torch.zeros((), device=A.device)
    loss = torch.where(kept, terms * weight, zero).double().sum().float().view(1)
    grad = _row_gradient(p, targets, kept, weight * dterm / case["temperature"], logits.dtype)
    return loss, logp, grad


# ---- the framework's operators --------------------------------------------------------------------------------------------

def _run_own(st):
    from metal_candle_b200 import training as F

    case, logits = st["case"], st["logits"]
    kind = case["kind"]
    if kind == "distill":
        return F.distillation_loss(logits, st["teacher_ids"], st["teacher_logits"], mask=st["mask"], temperature=case["temperature"],
                                   return_grad=True)
    targets = st["targets"]
    if kind in ("score", "logprob"):
        logp, lse = F.token_log_probs(logits, targets, ignore_index=IGNORE, temperature=case["temperature"])
        if kind == "score":
            return logp, lse
        return logp, F.token_log_probs_backward(logits, targets, logp, lse, st["dlogp"], ignore_index=IGNORE, temperature=case["temperature"])
    if kind == "preference":
        out = F.preference_loss(logits, targets, st["ref"], beta=0.1, label_smoothing=case["smoothing"], average_log_probs=case["average"],
                                ignore_index=IGNORE, return_grad=True)
        return out.loss, out.log_probs, out.grad
    out = F.policy_loss(logits, targets, st["advantages"], old_log_probs=st["old"], ref_log_probs=st["ref"], clip_low=0.2, clip_high=0.2,
                        kl_coef=case["kl"], temperature=case["temperature"], sequence_mean=case["sequence_mean"], ignore_index=IGNORE,
                        return_grad=True)
    return out.loss, out.log_probs, out.grad


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in float64 --------------------------------------------------------------------------------------------

def _exact_rows(case, logits, fn):
    """fn(first row, y) over the rows y = x / T [.., V] of the logits in float64, a part at a time."""
    x2 = logits.view(-1, logits.shape[-1])
    step = max(1, (1 << 26) // x2.shape[1])
    return [fn(i, x2[i:i + step].double() / case.get("temperature", 1.0)) for i in range(0, x2.shape[0], step)]


def exact(case, seed):
    st = prepare(case, seed)
    logits, kind = st["logits"], case["kind"]
    B, S, V = logits.shape
    M, T = B * S, case.get("temperature", 1.0)
    f64 = torch.float64
    if kind == "distill":
        ids, t = st["teacher_ids"].view(M, -1), st["teacher_logits"].view(M, -1).double() / T
        kept = st["mask"].view(M).to(f64)
        share = kept / max(1.0, float(kept.sum()))
        grad, loss = torch.empty(M, V, dtype=f64, device=logits.device), []

        def part(i, y):
            k = slice(i, i + y.shape[0])
            logp = torch.log_softmax(y, -1)
            logq = torch.log_softmax(t[k], -1)
            loss.append((logq.exp() * (logq - logp.gather(1, ids[k]))).sum(1) @ share[k] * T * T)
            g = logp.exp().scatter_add(1, ids[k], -logq.exp())
            grad[k] = g * (T * share[k])[:, None]

        _exact_rows(case, logits, part)
        return sum(loss).view(1), grad.view(B, S, V)
    targets = st["targets"].view(M)
    kept = targets != IGNORE
    tgt = torch.where(kept, targets, torch.zeros_like(targets))
    logp, lse = torch.zeros(M, dtype=f64, device=logits.device), torch.zeros(M, dtype=f64, device=logits.device)

    def stats(i, y):
        k = slice(i, i + y.shape[0])
        z = torch.logsumexp(y, -1)
        lse[k] = z
        logp[k] = y[torch.arange(y.shape[0], device=y.device), tgt[k]] - z

    _exact_rows(case, logits, stats)
    logp, keep64 = torch.where(kept, logp, logp * 0), kept.to(f64)

    def gradient(dlogp):
        """From d loss / d logp of every position."""
        grad = torch.empty(M, V, dtype=f64, device=logits.device)

        def part(i, y):
            k = slice(i, i + y.shape[0])
            c = (dlogp[k] * keep64[k] / T)[:, None]
            grad[k] = -c * torch.softmax(y, -1)
            grad[k].scatter_add_(1, tgt[k, None], c)

        _exact_rows(case, logits, part)
        return grad.view(B, S, V)

    if kind == "score":
        return logp.view(B, S), (lse * keep64).view(B, S)
    if kind == "logprob":
        return logp.view(B, S), gradient(st["dlogp"].double().view(M))
    leaf = logp.clone().requires_grad_(True)   # the rest of the loss is a handful of numbers a token: differentiated by autograd
    table, keep_bs = leaf.view(B, S), keep64.view(B, S)
    if kind == "preference":
        P, eps = case["pairs"], case["smoothing"]
        sums = (table * keep_bs).sum(1)
        if case["average"]:
            sums = sums / keep_bs.sum(1).clamp_min(1)
        away = sums - st["ref"].double()
        z = 0.1 * (away[:P] - away[P:])
        loss = -((1 - eps) * torch.nn.functional.logsigmoid(z) + eps * torch.nn.functional.logsigmoid(-z)).mean()
        loss.backward()
        return loss.detach().view(1), sums.detach(), gradient(leaf.grad)
    A = st["advantages"].double()
    A = A if A.dim() == 2 else A.view(B, 1)
    ratio = torch.exp(table - st["old"].double())
    term = -torch.min(ratio * A, torch.clamp(ratio, 0.8, 1.2) * A)
    if case["kl"] > 0:
        away = st["ref"].double() - table
        term = term + case["kl"] * (torch.exp(away) - away - 1)
    if case["sequence_mean"]:
        n = keep_bs.sum(1)
        loss = ((term * keep_bs).sum(1) / n.clamp_min(1)).sum() / (n > 0).sum().clamp_min(1)
    else:
        loss = (term * keep_bs).sum() / keep_bs.sum().clamp_min(1)
    loss.backward()
    return loss.detach().view(1), logp.view(B, S), gradient(leaf.grad)
