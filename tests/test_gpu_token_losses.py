"""GPU: the losses over given tokens and their gradients against their definitions in float64.

Tolerances, for all of them: exponents are differences of logits times log2(e) / T, rounded three times (2^-24 each) of at
most some 60, and an exponential has an error of 2^-22: 1e-5 for any probability that matters and 2e-5 for a sum of 150000
of them in float32, so logp is good to 2e-5 + 1e-6 |logp| (a float32 value's own rounding and that of d ln 2 are 2^-24 each of
it).  A gradient is a row coefficient times (onehot - p): relative 5e-5 of each, with what the coefficient's own exponentials
make of logp's error, and rounded to its type once, half a step (eps / 2).
"""
import math

import pytest
import torch

from metal_candle_b200 import _lib
from metal_candle_b200 import training as F

pytestmark = pytest.mark.gpu

IGN = -100
BF, F32 = torch.bfloat16, torch.float32


def half(dtype):
    return torch.finfo(dtype).eps / 2


def make(dev, B, S, V, dtype, seed=0, keep=0.7, tdtype=torch.int64):
    g = torch.Generator(device=dev).manual_seed(1000 * seed + V + S)
    x = (torch.randn(B, S, V, device=dev, generator=g) * 2.5)
    t = torch.randint(0, V, (B, S), device=dev, generator=g)
    x.scatter_add_(2, t[..., None], 10 * torch.rand(B, S, 1, device=dev, generator=g))
    t = torch.where(torch.rand(B, S, device=dev, generator=g) < keep, t, torch.full_like(t, IGN))
    return x.to(dtype), t.to(tdtype), g


def rows64(x, t, T=1.0):
    """log-probabilities (0 where left out), probabilities and the mask, in float64."""
    y = x.double() / T
    lse = torch.logsumexp(y, -1)
    kept = (t != IGN) & (t != -1)
    logp = y.gather(-1, t.long().clamp(0, x.shape[-1] - 1)[..., None])[..., 0] - lse
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    return torch.where(kept, logp, zero), torch.where(kept, lse, zero), torch.softmax(y, -1), kept


def grad64(p, t, kept, coef):
    """coef (onehot - p) and the size of its parts."""
    hot = torch.zeros_like(p).scatter_(-1, t.long().clamp_min(0)[..., None], 1.0)
    c = torch.where(kept, coef, torch.zeros_like(coef))[..., None]
    return c * (hot - p), c.abs() * (hot - p).abs()


def check_logp(got, want):
    assert ((got.double() - want).abs() <= 2e-5 + 1e-6 * want.abs()).all(), float((got.double() - want).abs().max())


def check_grad(got, want, spread, scale=5e-5):
    """`spread`: what the relative error of the parts comes to in an element."""
    tol = half(got.dtype) * want.abs() + scale * spread + 1e-36
    worst = ((got.double() - want).abs() - tol).max()
    assert worst <= 0, float(worst)


SHAPES = [(1, 1, 1), (2, 3, 2), (1, 1, 17), (2, 5, 50), (2, 7, 1000), (4, 33, 2050), (2, 3, 8193), (2, 4, 32000), (2, 3, 50257), (2, 2, 151936),
          (2, 1, 420001), (2, 2, 700001)]   # the last: longer than the one-pass kernel's rows
both = pytest.mark.parametrize("dtype", [F32, BF])
shapes = pytest.mark.parametrize("B,S,V", SHAPES)


@both
@shapes
@pytest.mark.parametrize("T,tdtype", [(1.0, torch.int64), (0.7, torch.int32)])
def test_token_log_probs(cuda_device, dtype, B, S, V, T, tdtype):
    x, t, g = make(cuda_device, B, S, V, dtype, 1, tdtype=tdtype)
    keep = x.clone()
    logp, lse = F.token_log_probs(x, t, ignore_index=IGN, temperature=T)
    want, wlse, p, kept = rows64(x, t, T)
    assert torch.equal(x, keep)
    check_logp(logp, want)
    check_logp(lse, wlse)
    assert (logp[~kept] == 0).all() and (lse[~kept] == 0).all()
    d = torch.randn(B, S, device=cuda_device, generator=g)
    grad = F.token_log_probs_backward(x, t, logp, lse, d, ignore_index=IGN, temperature=T)
    assert grad.shape == x.shape and grad.dtype == dtype and torch.equal(x, keep)
    wg, spread = grad64(p, t, kept, d.double() / T)
    check_grad(grad, wg, 2 * spread)   # lse and each exponential
    assert (grad[~kept] == 0).all()


def policy64(logp, kept, A, old, ref, lo, hi, kl, seq_mean):
    leaf = logp.clone().requires_grad_(True)
    A = A.double() if A.dim() == 2 else A.double()[:, None]
    r = torch.exp(leaf - (old.double() if old is not None else leaf.detach()))
    rc = r.clamp(1 - lo, 1 + hi)
    term = -torch.minimum(r * A, rc * A)
    bound = torch.where(A >= 0, r > 1 + hi, r < 1 - lo).double()
    k = torch.zeros_like(leaf)
    if ref is not None:
        d = ref.double() - leaf
        k = torch.exp(d) - d - 1
        term = term + kl * k
    m = kept.double()
    n = m.sum(1, keepdim=True)
    w = m / n.clamp_min(1) / (n > 0).sum().clamp_min(1) if seq_mean else m / m.sum().clamp_min(1)
    loss = (w * term).sum()
    loss.backward()
    size = ((r * A).abs() + kl * (ref is not None) * (2 + k)).detach()   # of the parts of a token's term and of its derivative
    return loss.detach(), (w * k).sum().detach(), (w * bound).sum().detach(), leaf.grad, w, size


@both
@shapes
@pytest.mark.parametrize("variant", range(6))
def test_policy_loss(cuda_device, dtype, B, S, V, variant):
    T, kl, seq_mean, per_token, with_old, with_ref = [(1.0, 0.0, False, False, True, False), (1.0, 0.04, True, False, True, True),
                                                      (0.7, 0.2, False, True, True, True), (1.3, 0.0, True, True, False, False),
                                                      (1.0, 0.0, False, False, False, True), (1.0, 0.1, True, True, False, True)][variant]
    x, t, g = make(cuda_device, B, S, V, dtype, 2 + variant, keep=[0.7, 1.0][variant % 2])
    if B > 1:
        t[1] = IGN   # a sequence that keeps nothing
    logp, lse, p, kept = rows64(x, t, T)
    rnd = lambda *s: torch.randn(*s, device=cuda_device, generator=g)  # noqa: E731
    A = rnd(B, S) if per_token else rnd(B)
    drift = rnd(B, S) * 0.3
    for border in (0.8, 1.3):
        drift = torch.where((drift.exp() - border).abs() < 2e-3, drift + 1e-2, drift)   # on either side of a border both are right
    old = (logp - drift).float() if with_old else None
    ref = (logp + 0.5 * rnd(B, S)).float() if with_ref else None
    out = F.policy_loss(x, t, A, old, ref, clip_low=0.2, clip_high=0.3, kl_coef=kl, temperature=T, sequence_mean=seq_mean, ignore_index=IGN,
                        return_grad=True)
    wl, wk, wc, dlogp, w, size = policy64(logp, kept, A, old, ref, 0.2, 0.3, kl, seq_mean)
    check_logp(out.log_probs, logp)
    # logp's error of 2e-5 + 1e-6 |logp|, times what a term changes with logp
    slack = (w * size * (3e-5 + 1e-6 * logp.abs())).sum() + 1e-6 * wl.abs()
    assert abs(float(out.loss) - float(wl)) <= float(slack) + 1e-12
    assert abs(float(out.kl) - float(wk)) <= 1e-5 + 1e-4 * float(wk)
    assert abs(float(out.clip_fraction) - float(wc)) <= 1e-6
    wg, _ = grad64(p, t, kept, dlogp / T)
    _, spread = grad64(p, t, kept, w * size / T)
    check_grad(out.grad, wg, spread, 2e-4)
    plain = F.policy_loss(x, t, A, old, ref, clip_low=0.2, clip_high=0.3, kl_coef=kl, temperature=T, sequence_mean=seq_mean, ignore_index=IGN)
    assert plain.grad is None
    assert abs(float(plain.loss) - float(wl)) <= float(slack) + 1e-12


@both
@shapes
@pytest.mark.parametrize("eps,average", [(0.0, False), (0.1, True), (0.5, False)])
def test_preference_loss(cuda_device, dtype, B, S, V, eps, average):
    B += B % 2
    x, t, g = make(cuda_device, B, S, V, dtype, 11)
    t[B // 2] = IGN   # a rejected answer of no tokens
    logp, lse, p, kept = rows64(x, t)
    n = kept.sum(1).clamp_min(1) if average else torch.ones(B, device=cuda_device)
    leaf = logp.clone().requires_grad_(True)
    sums = (leaf * kept).sum(1) / n
    ref = (sums.detach() + torch.randn(B, device=cuda_device, generator=g)).float()
    P, beta = B // 2, 0.3
    away = sums - ref.double()
    z = beta * (away[:P] - away[P:])
    ls = torch.nn.functional.logsigmoid
    loss = -((1 - eps) * ls(z) + eps * ls(-z)).mean()
    loss.backward()
    out = F.preference_loss(x, t, ref, beta=beta, label_smoothing=eps, average_log_probs=average, ignore_index=IGN, return_grad=True)
    err = (2e-5 * kept.sum(1) + 1e-6 * (logp * kept).abs().sum(1)) / n + 1e-6 * sums.detach().abs()   # of a sequence's sum
    assert ((out.log_probs.double() - sums.detach()).abs() <= err).all()
    zerr = beta * float((err + 1e-6 * ref.abs()).max()) * 2
    assert abs(float(out.loss) - loss.item()) <= zerr + 1e-6
    wg, spread = grad64(p, t, kept, leaf.grad)
    # d loss / d z = eps - sigma(-z), off by at most a quarter of z's error
    _, more = grad64(p, t, kept, (beta / P / n)[:, None].expand(B, S).double())
    check_grad(out.grad, wg, spread * 2 + more * (zerr / 4 + 1e-6) / 5e-5)
    assert F.preference_loss(x, t, ref, beta=beta, ignore_index=IGN).grad is None


def teacher(dev, g, B, S, V, K, dtype):
    ids = torch.stack([torch.randperm(V, device=dev, generator=g)[:K] for _ in range(B * S)]).view(B, S, K)
    return ids, (torch.randn(B, S, K, device=dev, generator=g) * 3).to(dtype)


def distill64(x, ids, tl, mask, T):
    leaf = x.double().requires_grad_(True)
    logp = torch.log_softmax(leaf / T, -1)
    logq = torch.log_softmax(tl.double() / T, -1)
    q = logq.exp()
    kl = torch.where(q > 0, q * (logq - logp.gather(-1, ids.long().clamp(0, x.shape[-1] - 1))), torch.zeros_like(q)).sum(-1)
    w = mask.double() / mask.sum().clamp_min(1)
    loss = (w * T * T * kl).sum()
    loss.backward()
    parts = logp.exp().detach().scatter_add(-1, ids.long().clamp(0, x.shape[-1] - 1), q) * (w * T)[..., None]
    size = (w * T * T * (1 + (q * (logq.nan_to_num(0, 0, 0).abs())).sum(-1) + kl.abs())).sum().detach()
    return loss.detach(), leaf.grad, parts, float(size)


@both
@pytest.mark.parametrize("B,S,V,K", [(1, 1, 1, 1), (2, 3, 2, 2), (1, 2, 17, 5), (2, 5, 50, 50), (2, 7, 1000, 64), (3, 11, 2050, 33), (2, 3, 8193, 257),
                                     (2, 4, 32000, 1024), (2, 3, 50257, 101), (2, 2, 151936, 64), (1, 2, 420001, 8),
                                     (2, 2, 700001, 40)])
@pytest.mark.parametrize("T,tdtype,masked", [(1.0, None, False), (2.0, F32, True), (0.5, BF, True)])
def test_distillation_loss(cuda_device, dtype, B, S, V, K, T, tdtype, masked):
    x, t, g = make(cuda_device, B, S, V, dtype, 5)
    ids, tl = teacher(cuda_device, g, B, S, V, K, tdtype or dtype)
    mask = torch.rand(B, S, device=cuda_device, generator=g) < 0.6
    mask[0, 0] = True
    m = mask if masked else torch.ones_like(mask)
    if masked:
        ids = ids.to(torch.int32)
    loss, grad = F.distillation_loss(x, ids, tl, mask=mask if masked else None, temperature=T, return_grad=True)
    wl, wg, parts, size = distill64(x, ids, tl, m, T)
    assert abs(float(loss) - float(wl)) <= 3e-5 * size
    check_grad(grad, wg, parts)
    assert (grad[~m] == 0).all()
    assert torch.equal(F.distillation_loss(x, ids, tl, mask=(mask.to(torch.uint8) * 3) if masked else None, temperature=T), loss)


@both
@pytest.mark.parametrize("V", [60, 5000, 151936])
def test_teacher_entries_that_repeat_or_count_for_nothing(cuda_device, dtype, V):
    B, S, K = 2, 4, 48
    x, t, g = make(cuda_device, B, S, V, dtype, 6)
    ids, tl = teacher(cuda_device, g, B, S, V, K, F32)
    ids[0, 0, 1:] = ids[0, 0, 0]                 # one id throughout
    ids[0, 1, 8:40] = ids[0, 1, :32].clone()             # in pairs
    ids[0, 2, 5] = ids[0, 2, 40]
    tl[0, 3, 1:] = -math.inf                     # one entry is left: cross-entropy
    ids[0, 3, 1:] = -7                           # ... whose companions name nothing
    tl[1, 0, ::2] = -math.inf
    ids[1, 0, ::2] = V + 3
    tl[1, 1] = torch.finfo(F32).min              # uniform over its entries
    tl[1, 2, 3:] = torch.finfo(F32).min          # three are left
    mask = torch.ones(B, S, dtype=torch.bool, device=cuda_device)
    loss, grad = F.distillation_loss(x, ids, tl, temperature=1.5, return_grad=True)
    tl64 = tl.double()
    tl64[1, 1] = 0
    wl, wg, parts, size = distill64(x, ids, tl64, mask, 1.5)
    assert abs(float(loss) - float(wl)) <= 3e-5 * size
    check_grad(grad, wg, parts)
    again = F.distillation_loss(x, ids, tl, temperature=1.5, return_grad=True)
    assert torch.equal(again[0], loss) and torch.equal(again[1], grad)
    # a position whose entries are all -inf adds nothing, and still counts in the mean
    tl[1, 3] = -math.inf
    loss2, grad2 = F.distillation_loss(x, ids, tl, temperature=1.5, return_grad=True)
    assert (grad2[1, 3] == 0).all() and torch.equal(grad2[:, :3], grad[:, :3])
    lone = F.distillation_loss(x[1:, 3:], ids[1:, 3:], (tl64[1:, 3:]).float(), temperature=1.5)
    assert abs(float(loss2) + float(lone) / (B * S) - float(loss)) <= 1e-5 * size


@both
@pytest.mark.parametrize("V", [50, 5000, 8193, 50257, 151936])
def test_masked_and_extreme_logits(cuda_device, dtype, V):
    from tests.test_gpu_extreme_values import masked_logits

    x = masked_logits(V, dtype, cuda_device)
    x = torch.cat([x, x[:2].clone()]).view(1, 10, V)
    t = torch.ones(1, 10, dtype=torch.int64, device=cuda_device)
    x[0, 8, 1] = -math.inf                       # the target itself is masked
    x[0, 9] = -math.inf
    x[0, 9, 1] = 3.0                             # nothing but the target is left
    d = torch.ones(1, 10, device=cuda_device)
    logp, lse = F.token_log_probs(x, t)
    grad = F.token_log_probs_backward(x, t, logp, lse, d)
    fused = F.policy_loss(x, t, torch.full((1,), 10.0, device=cuda_device), return_grad=True)
    dl, dg = F.distillation_loss(x, t.view(1, 10, 1), torch.zeros(1, 10, 1, device=cuda_device), return_grad=True)
    for i in range(10):
        r = x[0, i].double()
        if r.isnan().any():
            for out in (logp[0, i], grad[0, i], fused.log_probs[0, i], fused.grad[0, i], dg[0, i]):
                assert out.isnan().all(), i
            continue
        z = r - r.max()
        lp = z - z.exp().sum().log()
        want = lp.exp().neg()
        want[1] += 1.0
        if i == 8:
            assert logp[0, i] == -math.inf and fused.log_probs[0, i] == -math.inf
        else:
            check_logp(logp[0, i], lp[1])
            check_logp(fused.log_probs[0, i], lp[1])
        check_grad(grad[0, i], want, want.abs())
        check_grad(fused.grad[0, i], -want, want.abs())   # ten positions, advantage 10: each counts once
        check_grad(dg[0, i], -want / 10, want.abs() / 10)
    assert _lib.device_status() == 0


def test_targets_that_name_nothing(cuda_device):
    """Out of range: NaN, there and in the loss, and nowhere else."""
    x, t, g = make(cuda_device, 4, 5, 300, BF, 7, keep=1.0)
    clean = F.policy_loss(x, t, torch.ones(4, device=cuda_device), ignore_index=IGN, return_grad=True)
    for bad in (300, -2, 1 << 40, -(1 << 40)):
        t2 = t.clone()
        t2[2, 3] = bad
        logp, lse = F.token_log_probs(x, t2, ignore_index=IGN)
        assert logp[2, 3].isnan() and logp.isnan().sum() == 1
        grad = F.token_log_probs_backward(x, t2, logp, lse, torch.ones_like(logp), ignore_index=IGN)
        assert grad[2, 3].isnan().all() and grad.isnan().sum() == 300
        out = F.policy_loss(x, t2, torch.ones(4, device=cuda_device), ignore_index=IGN, return_grad=True)
        assert out.loss.isnan() and out.grad[2, 3].isnan().all() and out.grad.isnan().sum() == 300
        assert torch.equal(out.grad[:2], clean.grad[:2])
        pref = F.preference_loss(x, t2, torch.zeros(4, device=cuda_device), ignore_index=IGN, return_grad=True)
        assert pref.loss.isnan() and pref.log_probs.isnan().tolist() == [False, False, True, False]
        assert not pref.grad[1].isnan().any() and not pref.grad[3].isnan().any()
    ids, tl = teacher(cuda_device, g, 4, 5, 300, 6, BF)
    ids[1, 2, 3] = 300
    loss, grad = F.distillation_loss(x, ids, tl, return_grad=True)
    assert loss.isnan() and grad[1, 2].isnan().all() and grad.isnan().sum() == 300


def test_nothing_kept(cuda_device):
    x, t, g = make(cuda_device, 2, 6, 1500, BF, 8)
    t.fill_(IGN)
    t[0, 0] = -1                                  # always left out, like the ignore index
    x[0, 1] = math.nan                            # what is left out is not looked at
    ids, tl = teacher(cuda_device, g, 2, 6, 1500, 4, BF)
    one = torch.ones(2, device=cuda_device)
    for seq_mean in (False, True):
        out = F.policy_loss(x, t, one, sequence_mean=seq_mean, ignore_index=IGN, return_grad=True)
        assert out.loss == 0 and out.kl == 0 and out.clip_fraction == 0 and (out.grad == 0).all() and (out.log_probs == 0).all()
    pref = F.preference_loss(x, t, torch.zeros(2, device=cuda_device), ignore_index=IGN, return_grad=True)
    assert abs(float(pref.loss) - math.log(2)) < 1e-6 and (pref.grad == 0).all()
    loss, grad = F.distillation_loss(x, ids, tl, mask=torch.zeros(2, 6, dtype=torch.bool, device=cuda_device), return_grad=True)
    assert loss == 0 and (grad == 0).all()


def layouts(dev, B, S, V, dtype):
    """The same logits in other strides, alignments and orders."""
    x, t, g = make(dev, B, S, V, dtype, 9)
    pad = torch.randn(B, S, V + 13, device=dev, generator=g).to(dtype)
    pad[..., :V] = x
    wide = torch.randn(B, S, ((V + 7) // 8) * 8 + 64, device=dev, generator=g).to(dtype)
    wide[..., :V] = x
    shift = torch.randn(B, S + 1, V, device=dev, generator=g).to(dtype)
    shift[:, :S] = x
    flat = torch.empty(B * S * V + 3, dtype=dtype, device=dev)
    flat[1:1 + B * S * V] = x.reshape(-1)
    return x, t, g, [("padded vocabulary", pad[..., :V]), ("padded to vectors", wide[..., :V]), ("all but the last token", shift[:, :S]),
                     ("one element in", flat[1:1 + B * S * V].view(B, S, V)), ("tokens first", x.transpose(0, 1).contiguous().transpose(0, 1)),
                     ("vocabulary first", x.permute(2, 0, 1).contiguous().permute(1, 2, 0))]


@both
@pytest.mark.parametrize("V", [31, 1000, 2056, 50257, 151936])
def test_strides_and_alignments(cuda_device, dtype, V):
    B, S, K = 2, 3, 7
    x, t, g, views = layouts(cuda_device, B, S, V, dtype)
    ids, tl = teacher(cuda_device, g, B, S, V, K, dtype)
    A, old = torch.randn(B, S, device=cuda_device, generator=g), torch.randn(B, S, device=cuda_device, generator=g) * 0.1 - 3
    logp64, _, p, kept = rows64(x, t)
    d = torch.randn(B, S, device=cuda_device, generator=g)
    _, wpg, parts, size = distill64(x, ids, tl, torch.ones_like(kept), 1.0)
    _, _, _, dlogp, w, psize = policy64(logp64, kept, A, old, old, 0.2, 0.2, 0.1, False)
    for name, v in views:
        assert torch.equal(v, x), name
        logp, lse = F.token_log_probs(v, t, ignore_index=IGN)
        check_logp(logp, logp64)
        wg, spread = grad64(p, t, kept, d.double())
        check_grad(F.token_log_probs_backward(v, t, logp, lse, d, ignore_index=IGN), wg, 2 * spread)
        out = F.policy_loss(v, t, A.t().contiguous().t(), old, old, kl_coef=0.1, ignore_index=IGN, return_grad=True)
        wg, _ = grad64(p, t, kept, dlogp)
        _, spread = grad64(p, t, kept, w * psize)
        check_grad(out.grad, wg, spread, 2e-4)
        check_grad(F.distillation_loss(v, ids, tl, return_grad=True)[1], wpg, parts)
        pref = F.preference_loss(v, t, torch.zeros(B, device=cuda_device), ignore_index=IGN, return_grad=True)
        assert ((pref.log_probs.double() - logp64.sum(1)).abs() <= S * 2e-5 + 2e-6 * logp64.abs().sum(1)).all(), name


def run_all(x, t, g, V, K=9):
    B, S = t.shape
    ids, tl = teacher(x.device, g, B, S, V, K, x.dtype)
    A, old = torch.randn(B, device=x.device, generator=g), torch.randn(B, S, device=x.device, generator=g) * 0.1 - 3
    ref = torch.randn(B, device=x.device, generator=g)
    d = torch.randn(B, S, device=x.device, generator=g)
    torch.cuda.synchronize()

    def run():
        logp, lse = F.token_log_probs(x, t, ignore_index=IGN)
        out = [logp, lse, F.token_log_probs_backward(x, t, logp, lse, d, ignore_index=IGN)]
        out += F.policy_loss(x, t, A, old, old, kl_coef=0.1, sequence_mean=True, ignore_index=IGN, return_grad=True)
        out += F.preference_loss(x, t, ref, ignore_index=IGN, return_grad=True)
        out += F.distillation_loss(x, ids, tl, mask=t != IGN, temperature=2.0, return_grad=True)
        return out

    return run


def same(a, b):
    return all(torch.equal(u, v) for u, v in zip(a, b))


@both
@pytest.mark.parametrize("B,S,V", [(2, 100, 1000), (4, 50, 32000), (2, 37, 50257), (2, 200, 151936)])
def test_streams_graphs_and_repeated_calls(cuda_device, dtype, B, S, V):
    """Every sum has one order: the same results on every call, on other streams beside one another, captured and replayed."""
    works = [run_all(*make(cuda_device, B, S, V, dtype, s), V) for s in (1, 2)]
    want = [w() for w in works]
    torch.cuda.synchronize()
    assert all(same(w(), ref) for w, ref in zip(works, want))
    streams = [torch.cuda.Stream() for _ in works]
    got = [[], []]
    for _ in range(4):
        for i, (w, s) in enumerate(zip(works, streams)):
            with torch.cuda.stream(s):
                got[i].append(w())
    torch.cuda.synchronize()
    assert all(same(out, ref) for runs, ref in zip(got, want) for out in runs)
    del got
    graphs, outs = [], []
    for w in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(w())
        graphs.append(graph)
    for _ in range(3):
        for o in outs:
            for v in o:
                v.fill_(-3)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        works[0]()
        torch.cuda.synchronize()
        assert all(same(o, ref) for o, ref in zip(outs, want))
    assert _lib.device_status() == 0


def test_infinite_divergence_that_is_only_reported(cuda_device):
    """kl_coef = 0: a reference that is infinitely far away is seen in `kl` and nowhere else."""
    x, t, g = make(cuda_device, 2, 3, 100, F32, 16, keep=1.0)
    A, ref = torch.ones(2, device=cuda_device), torch.zeros(2, 3, device=cuda_device)
    ref[0, 1] = 500.0
    far = F.policy_loss(x, t, A, None, ref, return_grad=True)
    near = F.policy_loss(x, t, A, None, None, return_grad=True)
    assert far.kl == math.inf and torch.equal(far.loss, near.loss) and torch.equal(far.grad, near.grad)


def test_long_sequences_of_pairs(cuda_device):
    """Sums of many tokens: 9001 log-probabilities a sequence, each good to 2e-5 + 1e-6 |logp| (three logits each, so below 12)."""
    x, t, g = make(cuda_device, 2, 9001, 3, F32, 17, keep=0.9)
    logp, _, _, kept = rows64(x, t)
    for average in (False, True):
        n = kept.sum(1) if average else torch.ones(2, device=cuda_device)
        out = F.preference_loss(x, t, (logp.sum(1) / n).float(), average_log_probs=average, ignore_index=IGN)
        assert ((out.log_probs.double() - logp.sum(1) / n).abs() <= (9001 * 3.2e-5 + 1e-6 * logp.sum(1).abs()) / n).all()


def test_first_calls_are_captured(cuda_device):
    """In a process of its own: nothing that a first call sets up is forbidden under capture."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from metal_candle_b200 import _lib
from metal_candle_b200 import training as F
_lib.init(0)
dev = torch.device("cuda", 0)
cases = []
for V in (500, 40000, 151936):
    for dt in (torch.bfloat16, torch.float32):
        x = torch.randn(2, 6, V, device=dev).to(dt)
        t = torch.randint(0, V, (2, 6), device=dev)
        cases.append((x, t, torch.randn(2, device=dev), torch.rand(2, 6, 4, device=dev).argsort(-1), torch.randn(2, 6, 4, device=dev)))
def run(x, t, a, ids, tl):
    logp, lse = F.token_log_probs(x, t)
    return [logp, F.token_log_probs_backward(x, t, logp, lse, logp), *F.policy_loss(x, t, a, return_grad=True),
            *F.preference_loss(x, t, a, return_grad=True), *F.distillation_loss(x, ids, tl, return_grad=True)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = [run(*c) for c in cases]
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(u, v) for c, out in zip(cases, captured) for u, v in zip(run(*c), out))
assert _lib.device_status() == 0
print("captured")
"""
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("M,V", [(14402, 151936), (2200002, 1000)])
def test_offsets_past_32_bits(cuda_device, M, V):
    """2.2e9 elements of logits and of their gradient: rows at both ends and where a 32-bit offset would turn over."""
    if torch.cuda.mem_get_info(cuda_device)[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    g = torch.Generator(device=cuda_device).manual_seed(11)
    x = torch.empty(1, M, V, dtype=BF, device=cuda_device)
    for part in x[0].split((1 << 28) // V):
        part.copy_(2.5 * torch.randn(part.shape, device=cuda_device, generator=g))
    t = torch.randint(0, V, (1, M), device=cuda_device, generator=g)
    turn = 2 ** 31 // V
    rows = torch.tensor([0, 1, turn - 1, turn, turn + 1, M - 2, M - 1], device=cuda_device)
    logp, lse, p, kept = rows64(x[:, rows], t[:, rows])

    def check(grad, coef, spread):
        wg, size = grad64(p, t[:, rows], kept, coef)
        check_grad(grad[:, rows], wg, spread * size)

    got, glse = F.token_log_probs(x, t)
    check_logp(got[:, rows], logp)
    d = torch.randn(1, M, device=cuda_device, generator=g)
    check(F.token_log_probs_backward(x, t, got, glse, d), d[:, rows].double(), 2)
    A = torch.randn(1, M, device=cuda_device, generator=g)
    out = F.policy_loss(x, t, A, return_grad=True)
    check_logp(out.log_probs[:, rows], logp)
    check(out.grad, -A[:, rows].double() / M, 2)
    del out
    pair = F.preference_loss(x.view(2, M // 2, V), t.view(2, M // 2), torch.zeros(2, device=cuda_device), beta=1e-4, return_grad=True)
    z = 1e-4 * (got[0, :M // 2].double().sum() - got[0, M // 2:].double().sum())
    # each of M log-probabilities is good to 2e-5 + 1e-6 |logp|, and the derivative of sigma is at most 1/4
    assert abs(float(pair.loss) - math.log1p(math.exp(-float(z)))) <= 1e-4 * M * 4e-5 + 1e-6
    c = 1e-4 * (torch.sigmoid(z) - 1)
    sign = torch.where(rows < M // 2, 1.0, -1.0).double()[None]
    check(pair.grad.view(1, M, V), c * sign, 2 + 1e-4 * M * 4e-5 / 5e-5)
    del pair
    ids = torch.randint(0, V, (1, M, 4), device=cuda_device, generator=g)
    tl = torch.randn(1, M, 4, device=cuda_device, generator=g)
    loss, grad = F.distillation_loss(x, ids, tl, return_grad=True)
    wl, wg, parts, size = distill64(x[:, rows], ids[:, rows], tl[:, rows], torch.ones_like(rows, dtype=torch.bool)[None], 1.0)
    n = len(rows) / M   # distill64 has the mean of these rows
    check_grad(grad[:, rows], wg * n, parts * n)
    assert math.isfinite(float(loss))


def test_gradients_against_differences(cuda_device):
    """d loss along a direction, against (loss(x + h u) - loss(x - h u)) / 2h of the same entry points in float32: h = 0.02 along a
    direction of unit length; the third derivative of these losses along it is below 10 (0.0007 in the quotient), a loss
    below 4 is off by at most 2e-6 (1e-4)."""
    B, S, V, K = 2, 3, 40, 6
    x, t, g = make(cuda_device, B, S, V, F32, 12, keep=1.0)
    ids, tl = teacher(cuda_device, g, B, S, V, K, F32)
    rnd = lambda *s: torch.randn(*s, device=cuda_device, generator=g)  # noqa: E731
    A, old, ref, sref = rnd(B), F.token_log_probs(x, t)[0] + 0.05, F.token_log_probs(x, t)[0] + 0.3 * rnd(B, S), rnd(B)

    losses = {
        "policy": lambda y, grad=False: F.policy_loss(y, t, A, old, ref, kl_coef=0.2, temperature=1.2, clip_low=0.9, clip_high=3.0, return_grad=grad),
        "preference": lambda y, grad=False: F.preference_loss(y, t, sref, beta=0.5, label_smoothing=0.1, return_grad=grad),
        "distill": lambda y, grad=False: F.distillation_loss(y, ids, tl, temperature=1.5, return_grad=True),
    }
    for name, f in losses.items():
        grad = f(x, True)[-1].double()
        for _ in range(4):
            u = rnd(B, S, V)
            u = u / u.norm()
            h = 0.02
            diff = (float(f(x + h * u)[0].double()) - float(f(x - h * u)[0].double())) / (2 * h)
            along = float((grad * u.double()).sum())
            assert abs(diff - along) <= 1e-3, (name, diff, along)
        # along the gradient itself the quotient is its length
        u = (grad / grad.norm()).float()
        diff = (float(f(x + 0.02 * u)[0].double()) - float(f(x - 0.02 * u)[0].double())) / 0.04
        assert abs(diff - float(grad.norm())) <= 1e-3, name


def test_gradients_in_place(cuda_device):
    """The C entry points write the gradient over the logits."""
    import ctypes as C

    for dtype in (F32, BF):
        for V in (1000, 2049, 50257, 151936):
            B, S, K = 2, 5, 12
            x, t, g = make(cuda_device, B, S, V, dtype, 13)
            ids, tl = teacher(cuda_device, g, B, S, V, K, dtype)
            A = torch.randn(B, S, device=cuda_device, generator=g)
            lib = _lib.load()
            want_p = F.policy_loss(x, t, A, ignore_index=IGN, return_grad=True)
            want_d = F.distillation_loss(x, ids, tl, return_grad=True)
            logp, lse = F.token_log_probs(x, t, ignore_index=IGN)
            want_b = F.token_log_probs_backward(x, t, logp, lse, A, ignore_index=IGN)
            unit = F.token_log_probs_backward(x, t, logp, lse, torch.ones_like(A), ignore_index=IGN)
            rows = lambda y: C.byref(_lib.TokenLogits(y.data_ptr(), B, S, V, S * V, V, 1.0, int(dtype == BF)))  # noqa: E731
            tt = C.byref(_lib.TokenTargets(t.data_ptr(), 8, 1, IGN))
            ws = torch.empty(lib.mcb_token_loss_workspace_bytes(B, S), dtype=torch.uint8, device=cuda_device)
            st = torch.cuda.current_stream().cuda_stream
            y, lp, out = x.clone(), torch.empty(B, S, device=cuda_device), torch.empty(3, device=cuda_device)
            _lib.check(lib.mcb_policy_loss(rows(y), tt, C.byref(_lib.PolicyTerms(A.data_ptr(), 1, None, None, 0.2, 0.2, 0.0, 0)), 0, lp.data_ptr(),
                                           out.data_ptr(), y.data_ptr(), ws.data_ptr(), ws.numel(), st))
            assert torch.equal(y, want_p.grad) and torch.equal(out[:1], want_p.loss) and torch.equal(lp, want_p.log_probs)
            y = x.clone()
            _lib.check(lib.mcb_distill_loss(rows(y), C.byref(_lib.TeacherTop(ids.data_ptr(), tl.data_ptr(), K, 8, int(dtype == BF))), None, out.data_ptr(),
                                            y.data_ptr(), ws.data_ptr(), ws.numel(), st))
            assert torch.equal(y, want_d[1]) and torch.equal(out[:1], want_d[0])
            y = x.clone()
            _lib.check(lib.mcb_token_logprob_bwd(rows(y), tt, logp.data_ptr(), lse.data_ptr(), A.data_ptr(), 1, y.data_ptr(), st))
            assert torch.equal(y, want_b)
            y = x.clone()
            _lib.check(lib.mcb_token_logprob_fwd(rows(y), tt, lp.data_ptr(), None, y.data_ptr(), st))
            check_logp(lp, logp.double())
            p = torch.softmax(x.double(), -1)
            wg, spread = grad64(p, t, t != IGN, torch.ones(B, S, dtype=torch.float64, device=cuda_device))
            check_grad(y, wg, 2 * spread)
            check_grad(unit, wg, 2 * spread)


@pytest.mark.parametrize("B,S", [(1, 1), (3, 700), (5, 1000), (1, 9001), (9001, 1), (3000, 3), (40, 2500), (1, 70001), (23, 3100)])
@pytest.mark.parametrize("keep", [0.0, 0.6, 1.0])
def test_weights_of_the_mean(cuda_device, B, S, keep):
    """By one block and by a cluster, targets kept in registers and read again, sequences counted in shared memory and one by one; and the
    loss over the same rows, which takes them in the order the kernel finds."""
    import ctypes as C

    lib, V, M = _lib.load(), 16, B * S
    g = torch.Generator(device=cuda_device).manual_seed(B + S)
    t = torch.randint(0, V, (B, S), device=cuda_device, generator=g)
    kept = torch.rand(B, S, device=cuda_device, generator=g) < keep
    if B > 2:
        kept[1] = False
    t = torch.where(kept, t, torch.full_like(t, -1)).to(torch.int32)
    for seq_mean in (0, 1):
        w = torch.full((B, S), math.nan, device=cuda_device)
        _lib.check(lib.mcb_loss_weights(C.byref(_lib.TokenTargets(t.data_ptr(), 4, 0, 0)), None, w.data_ptr(), B, S, V, seq_mean,
                                        torch.cuda.current_stream().cuda_stream))
        n = kept.sum(1, keepdim=True)
        want = kept.double() / (n.clamp_min(1) * (n > 0).sum().clamp_min(1) if seq_mean else kept.sum().clamp_min(1))
        assert ((w.double() - want).abs() <= 3 * 2.0 ** -24 * want).all()   # two divisions and their product
        m8 = kept.to(torch.uint8)
        w2 = torch.full_like(w, math.nan)
        _lib.check(lib.mcb_loss_weights(None, m8.data_ptr(), w2.data_ptr(), B, S, V, seq_mean, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(w, w2)
        x = torch.randn(B, S, V, device=cuda_device, generator=g)
        out = F.policy_loss(x, t, torch.ones(B, S, device=cuda_device), sequence_mean=bool(seq_mean), return_grad=True)
        assert abs(float(out.loss) + float(want.sum())) <= 1e-5
        logp = torch.log_softmax(x.double(), -1).gather(-1, t.long().clamp_min(0)[..., None])[..., 0]
        check_logp(out.log_probs, torch.where(kept, logp, torch.zeros_like(logp)))
        wg, spread = grad64(torch.softmax(x.double(), -1), t, kept, -want)
        check_grad(out.grad, wg, 2 * spread)
        dist, grad = F.distillation_loss(x, t.clamp_min(0)[..., None], torch.zeros(B, S, 1, device=cuda_device), mask=kept, return_grad=True)
        share = kept.double() / kept.sum().clamp_min(1)
        assert abs(float(dist) + float((share * logp).sum())) <= 1e-4
        wg, spread = grad64(torch.softmax(x.double(), -1), t, kept, -share)
        check_grad(grad, wg, 4 * spread + share[..., None] * torch.softmax(x.double(), -1))


@both
@pytest.mark.parametrize("V", [300, 2049, 32000, 151936])
def test_rows_of_a_chunk(cuda_device, dtype, V):
    """The stages for a caller that makes the logits a chunk at a time: the whole calls' results, in place too, and rows that are left
    out are not looked at.  How a row is split over the chip depends on how many there are, so the sums' order does: both sides
    are off by the tolerance above, a gradient by half a step each."""

    def agree(got, want):
        check_grad(got, want.double(), want.double().abs(), 1e-4 + half(dtype))

    import ctypes as C

    B, S, K = 3, 7, 6
    x, t, g = make(cuda_device, B, S, V, dtype, 15)
    ids, tl = teacher(cuda_device, g, B, S, V, K, dtype)
    t[0, 2] = IGN
    t[2] = IGN
    mask = t != IGN
    A = torch.randn(B, S, device=cuda_device, generator=g)
    want_p = F.policy_loss(x, t, A, sequence_mean=True, ignore_index=IGN, return_grad=True)
    want_d = F.distillation_loss(x, ids, tl, mask=mask, temperature=1.5, return_grad=True)
    x = torch.where(mask[..., None], x, torch.full_like(x, math.nan))
    lib, st, M = _lib.load(), torch.cuda.current_stream().cuda_stream, B * S
    code = int(dtype == BF)
    new = lambda *s: torch.empty(*s, device=cuda_device)  # noqa: E731
    targets = lambda c: C.byref(_lib.TokenTargets(t.view(M)[c:].data_ptr(), 8, 1, IGN))  # noqa: E731
    w = new(M)
    for in_place in (False, True):
        y = x.clone().view(M, V)
        to = y if in_place else torch.empty_like(y)
        _lib.check(lib.mcb_loss_weights(targets(0), None, w.data_ptr(), B, S, V, 1, st))
        logp, parts = new(M), []
        for c0, c1 in ((0, 4), (4, 5), (5, 15), (15, M)):
            rows = C.byref(_lib.TokenLogits(y[c0:].data_ptr(), 1, c1 - c0, V, (c1 - c0) * V, V, 1.0, code))
            parts.append(new(3, c1 - c0))
            _lib.check(lib.mcb_policy_loss_rows(rows, targets(c0), C.byref(_lib.PolicyTerms(A.view(M)[c0:].data_ptr(), 1, None, None, 0.2, 0.2, 0.0, 0)),
                                                w[c0:].data_ptr(), logp[c0:].data_ptr(), parts[-1].data_ptr(), to[c0:].data_ptr(), st))
        out, terms = new(3), torch.cat(parts, 1)
        _lib.check(lib.mcb_loss_sums(terms.data_ptr(), M, 3, out.data_ptr(), st))
        agree(to.view(B, S, V), want_p.grad)
        assert ((logp.view(B, S) - want_p.log_probs).abs() <= 4e-5 + 2e-6 * want_p.log_probs.abs()).all()
        assert abs(float(out[0]) - float(want_p.loss)) <= 1e-4
        y = x.clone().view(M, V)
        to = y if in_place else torch.empty_like(y)
        m8 = mask.to(torch.uint8)
        _lib.check(lib.mcb_loss_weights(None, m8.data_ptr(), w.data_ptr(), B, S, V, 0, st))
        parts = []
        for c0, c1 in ((0, 6), (6, 16), (16, M)):
            rows = C.byref(_lib.TokenLogits(y[c0:].data_ptr(), 1, c1 - c0, V, (c1 - c0) * V, V, 1.5, code))
            top = C.byref(_lib.TeacherTop(ids.view(M, K)[c0:].data_ptr(), tl.view(M, K)[c0:].data_ptr(), K, 8, code))
            parts.append(new(c1 - c0))
            _lib.check(lib.mcb_distill_loss_rows(rows, top, w[c0:].data_ptr(), parts[-1].data_ptr(), to[c0:].data_ptr(), st))
        terms = torch.cat(parts)
        _lib.check(lib.mcb_loss_sums(terms.data_ptr(), M, 1, out.data_ptr(), st))
        agree(to.view(B, S, V), want_d[1])
        assert abs(float(out[0]) - float(want_d[0])) <= 6e-5 * (1 + float(want_d[0]))


def test_another_current_stream_and_memory_around(cuda_device):
    """Nothing but the outputs is written: the bytes around a gradient that starts off a 16-byte boundary stay."""
    import ctypes as C

    for dtype in (F32, BF):
        for V in (37, 2051, 50257):
            B, S = 2, 3
            x, t, g = make(cuda_device, B, S, V, dtype, 14)
            n = B * S * V
            lib = _lib.load()
            logp, lse = F.token_log_probs(x, t, ignore_index=IGN)
            A = torch.ones(B, S, device=cuda_device)
            want = F.policy_loss(x, t, A, ignore_index=IGN, return_grad=True)
            for off in (0, 1, 3, 8):
                buf = torch.full((n + 40,), 7.0, dtype=dtype, device=cuda_device)
                rows = C.byref(_lib.TokenLogits(x.data_ptr(), B, S, V, S * V, V, 1.0, int(dtype == BF)))
                tt = C.byref(_lib.TokenTargets(t.data_ptr(), 8, 1, IGN))
                ws = torch.empty(lib.mcb_token_loss_workspace_bytes(B, S), dtype=torch.uint8, device=cuda_device)
                out = torch.empty(3, device=cuda_device)
                _lib.check(lib.mcb_policy_loss(rows, tt, C.byref(_lib.PolicyTerms(A.data_ptr(), 1, None, None, 0.2, 0.2, 0.0, 0)), 0, logp.data_ptr(),
                                               out.data_ptr(), buf[16 + off:].data_ptr(), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
                got = buf[16 + off:16 + off + n].view(B, S, V)
                check_grad(got, want.grad.double(), want.grad.double().abs() + 1e-9, 1e-2 if dtype == BF else 1e-4)
                assert (buf[:16 + off] == 7).all() and (buf[16 + off + n:] == 7).all()
                buf.fill_(7.0)
                _lib.check(lib.mcb_token_logprob_bwd(rows, tt, logp.data_ptr(), lse.data_ptr(), A.data_ptr(), 1, buf[16 + off:].data_ptr(),
                                                     torch.cuda.current_stream().cuda_stream))
                assert (buf[:16 + off] == 7).all() and (buf[16 + off + n:] == 7).all()
    assert _lib.device_status() == 0
