"""GPU: the losses over given tokens where rows, targets or layouts are out of the ordinary, against float64 at the tolerances of
ordinary rows (see test_gpu_token_losses)."""
import ctypes as C
import math

import pytest
import torch

from metal_candle_b200 import _lib
from metal_candle_b200 import training as F
from tests.test_gpu_token_losses import BF, F32, IGN, both, check_grad, check_logp, grad64, make, rows64, teacher

pytestmark = pytest.mark.gpu


@both
@pytest.mark.parametrize("V", [50, 5001, 50257])
@pytest.mark.parametrize("T", [0.7, 1.0, 1.5, 2.0])
def test_log_probabilities_of_the_lowest_values(cuda_device, dtype, V, T):
    """y_t - lse down to where float32 ends, though y_t log2(e) lies beyond.  Two roundings of relative 2^-24 each may carry a value
    across that end: within 1e-6 of it both are right."""
    g = torch.Generator(device=cuda_device).manual_seed(20)
    x = torch.randn(1, 9, V, device=cuda_device, generator=g).to(dtype)
    low, most = torch.finfo(dtype).min, torch.finfo(torch.float32).max
    x[0, 3:6] = 3e38
    x[0, 6:8] = low
    x[0, 8, 2:] = -1e38
    x[0, :, 1] = torch.tensor([low, -2.5e38, -math.inf, low, 0.0, 2e38, -math.inf, low, low], device=cuda_device).to(dtype)
    t = torch.ones(1, 9, dtype=torch.int64, device=cuda_device)
    y = x.double()
    top = y.amax(-1, keepdim=True)
    want = ((y - top)[..., 1] / T - ((y - top) / T).exp().sum(-1).log())
    outs = [F.token_log_probs(x, t, temperature=T)[0]]
    for grad in (False, True):
        outs.append(F.policy_loss(x, t, torch.zeros(1, device=cuda_device), temperature=T, return_grad=grad).log_probs)
    for got in outs:
        for v, w in zip(got[0].tolist(), want[0].tolist()):
            if w < -most * (1 - 1e-6):
                assert v == -math.inf or (w > -most * (1 + 1e-6) and v < -most * (1 - 2e-6)), (v, w)
            else:
                assert abs(v - w) <= 2e-5 + 1e-6 * abs(w), (v, w)


@both
@pytest.mark.parametrize("V", [50, 5000, 50257, 700001])
def test_policy_loss_of_nan_logits(cuda_device, dtype, V):
    """NaN in a row is seen in the loss too, when the ratio is 1 for want of old log-probabilities."""
    x, t, g = make(cuda_device, 2, 2, V, dtype, 28, keep=1.0)
    old = torch.zeros(2, 2, device=cuda_device)
    x[1, 0, (int(t[1, 0]) + 1) % V] = math.nan
    for grad in (False, True):
        for o in (None, old):
            out = F.policy_loss(x, t, torch.ones(2, device=cuda_device), o, return_grad=grad)
            assert out.loss.isnan() and out.log_probs.isnan().sum() == 1
    x[1, 0] = -math.inf     # nothing but the target, which is certain
    x[1, 0, int(t[1, 0])] = 1.0
    assert F.policy_loss(x, t, torch.ones(2, device=cuda_device)).loss == -1


@both
@pytest.mark.parametrize("V", [50, 5000, 50257, 151936, 700001])
def test_infinite_logits(cuda_device, dtype, V):
    """A logit that has overflowed makes its row NaN, at the target as in any other column, and no other row."""
    g = torch.Generator(device=cuda_device).manual_seed(22)
    x = torch.randn(2, 3, V, device=cuda_device, generator=g).to(dtype)
    t = torch.full((2, 3), 2, dtype=torch.int64, device=cuda_device)
    x[0, 1, 2] = math.inf       # the target
    x[1, 0, V // 2] = math.inf
    bad = torch.zeros(2, 3, dtype=torch.bool, device=cuda_device)
    bad[0, 1] = bad[1, 0] = True
    logp, lse = F.token_log_probs(x, t)
    outs = [F.token_log_probs_backward(x, t, logp, lse, torch.ones_like(logp)),
            F.policy_loss(x, t, torch.ones(2, device=cuda_device), return_grad=True).grad,
            F.distillation_loss(x, t[..., None], torch.zeros(2, 3, 1, device=cuda_device), return_grad=True)[1]]
    unit, lp = torch.empty_like(x), torch.empty_like(logp)
    rows = C.byref(_lib.TokenLogits(x.data_ptr(), 2, 3, V, 3 * V, V, 1.0, int(dtype == BF)))
    _lib.check(_lib.load().mcb_token_logprob_fwd(rows, C.byref(_lib.TokenTargets(t.data_ptr(), 8, 0, 0)), lp.data_ptr(), None, unit.data_ptr(),
                                                 torch.cuda.current_stream().cuda_stream))
    pol = F.policy_loss(x, t, torch.ones(2, device=cuda_device))
    for v in (logp, lse, lp, pol.log_probs):
        assert torch.equal(v.isnan(), bad)
    for v in outs + [unit]:
        assert torch.equal(v.isnan(), bad[..., None].expand(2, 3, V))
    assert pol.loss.isnan() and F.preference_loss(x, t, torch.zeros(2, device=cuda_device)).loss.isnan()


FAR = [-30.0, -100.0, -1e3, -1e4, -1e6, -1e9, None, -math.inf]   # None: the type's lowest value


def far_targets(dev, V, dtype, seed=21):
    """[1, rows, V], the target of every row column 1: of ordinary logits, of logits around 3e4 and of logits whose product with
    log2(e) overflows."""
    g = torch.Generator(device=dev).manual_seed(seed + V)
    n = len(FAR)
    x = torch.randn(1, 2 * n + 3, V, device=dev, generator=g) * 2.5
    x[0, n:2 * n] += 3e4
    x[0, 2 * n:] = 3e38
    x = x.to(dtype)
    for i, v in enumerate(FAR + FAR):
        x[0, i, 1] = torch.finfo(dtype).min if v is None else v
    x[0, 2 * n, 1] = -math.inf
    x[0, 2 * n + 1, 1] = 0.0
    x[0, 2 * n + 2, 1] = torch.finfo(dtype).min
    return x, torch.ones(x.shape[:2], dtype=torch.int64, device=dev), g


def in_place(x, t, logp, lse, d, T):
    """mcb_token_logprob_bwd over the logits."""
    B, S, V = x.shape
    y = x.clone()
    rows = C.byref(_lib.TokenLogits(y.data_ptr(), B, S, V, S * V, V, T, int(y.dtype == BF)))
    _lib.check(_lib.load().mcb_token_logprob_bwd(rows, C.byref(_lib.TokenTargets(t.data_ptr(), 8, 0, 0)), logp.data_ptr(), lse.data_ptr(),
                                                 d.data_ptr(), 1, y.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return y


def softmax64(x, T):
    """log-probabilities and probabilities with the largest logit taken out first, so that nothing overflows."""
    z = (x.double() - x.double().amax(-1, keepdim=True)) / T
    logp = z - z.exp().sum(-1, keepdim=True).log()
    return logp, logp.exp()


@both
@pytest.mark.parametrize("V", [50, 1000, 5001, 32000, 50257])
@pytest.mark.parametrize("T", [0.7, 1.0, 2.0])
def test_targets_far_below_the_rest(cuda_device, dtype, V, T):
    """A target that the present mask forbids (-1e4, -1e9, the type's lowest value), in the reverse pass: the other columns keep their
    softmax, at the tolerance of ordinary rows."""
    x, t, g = far_targets(cuda_device, V, dtype)
    d = torch.randn(t.shape, device=cuda_device, generator=g)
    logp, lse = F.token_log_probs(x, t, temperature=T)
    want, p = softmax64(x, T)
    most = torch.finfo(F32).max   # (what lies within roundings of float32's end may come out on either side of it)
    fits, beyond = want[..., 1] > -most * (1 - 1e-6), want[..., 1] < -most * (1 + 1e-6)
    assert ((logp.double() - want[..., 1])[fits].abs() <= 2e-5 + 1e-6 * want[..., 1][fits].abs()).all()
    assert (logp[beyond] == -math.inf).all()
    wg, spread = grad64(p, t, torch.ones_like(t, dtype=torch.bool), d.double() / T)
    check_grad(F.token_log_probs_backward(x, t, logp, lse, d, temperature=T), wg, 2 * spread)
    check_grad(in_place(x, t, logp, lse, d, T), wg, 2 * spread)


@both
@pytest.mark.parametrize("V", [50, 1000, 50257])
def test_pairs_with_targets_far_below_the_rest(cuda_device, dtype, V):
    """A chosen answer of one forbidden token against one of a likely token: z is so far below 0 that the coefficients are beta / pairs."""
    x, t, g = far_targets(cuda_device, V, dtype)
    P = t.shape[1]
    other = (torch.randn(P, 1, V, device=cuda_device, generator=g)).to(dtype)
    other[:, 0, 1] = 12.0
    x, t = torch.cat([x.view(P, 1, V), other]), torch.ones(2 * P, 1, dtype=torch.int64, device=cuda_device)
    out = F.preference_loss(x, t, torch.zeros(2 * P, device=cuda_device), beta=2.0, return_grad=True)
    _, p = softmax64(x, 1.0)
    c = torch.full((2 * P, 1), 2.0 / P, dtype=torch.float64, device=cuda_device)
    c[:P] *= -1
    wg, spread = grad64(p, t, torch.ones_like(t, dtype=torch.bool), c)
    check_grad(out.grad, wg, 2 * spread)
    assert out.loss == math.inf


def test_pairs_of_forbidden_tokens(cuda_device):
    """-inf at the target of a rejected answer: the pair is won for certain, a loss of 0 and no gradient; of a chosen one: an
    infinite loss, whose gradient is finite.  With smoothed labels either is infinite."""
    P, S, V, beta = 3, 2, 40, 0.5
    x, t, g = make(cuda_device, 2 * P, S, V, F32, 23, keep=1.0)
    ref = torch.zeros(2 * P, device=cuda_device)
    won, lost = x.clone(), x.clone()
    won[P + 1, 0, int(t[P + 1, 0])] = -math.inf
    lost[1, 0, int(t[1, 0])] = -math.inf
    out = F.preference_loss(won, t, ref, beta=beta, return_grad=True)
    alone = [F.preference_loss(won[[i, P + i]], t[[i, P + i]], ref[:2], beta=beta) for i in range(P)]
    assert float(alone[1].loss) == 0.0
    assert abs(float(out.loss) - (float(alone[0].loss) + float(alone[2].loss)) / P) <= 1e-6 * (1 + float(out.loss))
    assert (out.grad[[1, P + 1]] == 0).all() and not out.grad.isnan().any()
    assert F.preference_loss(won, t, ref, beta=beta, label_smoothing=0.1).loss == math.inf
    out = F.preference_loss(lost, t, ref, beta=beta, return_grad=True)
    assert out.loss == math.inf and out.grad.isfinite().all() and (out.grad[1] != 0).any()


@both
def test_strides_of_single_rows(cuda_device, dtype):
    """The stride of a dimension of one is any number: such logits are dense all the same, and may be written over."""
    lib, st = _lib.load(), torch.cuda.current_stream().cuda_stream
    for B, S, V in ((1, 5, 1001), (4, 1, 1001), (1, 1, 300), (1, 3, 50257)):
        x, t, g = make(cuda_device, B, S, V, dtype, 24, keep=1.0)
        logp, lse = F.token_log_probs(x, t)
        d = torch.randn(B, S, device=cuda_device, generator=g)
        _, _, p, kept = rows64(x, t)
        wg, spread = grad64(p, t, kept, d.double())
        strides = (7 if B == 1 else V if S == 1 else S * V, 5 if S == 1 else V)
        y = x.clone()
        rows = C.byref(_lib.TokenLogits(y.data_ptr(), B, S, V, *strides, 1.0, int(dtype == BF)))
        _lib.check(lib.mcb_token_logprob_bwd(rows, C.byref(_lib.TokenTargets(t.data_ptr(), 8, 0, 0)), logp.data_ptr(), lse.data_ptr(),
                                             d.data_ptr(), 1, y.data_ptr(), st))
        check_grad(y, wg, 2 * spread)
        y = x.clone()
        rows = C.byref(_lib.TokenLogits(y.data_ptr(), B, S, V, *strides, 1.0, int(dtype == BF)))
        lp = torch.empty_like(logp)
        _lib.check(lib.mcb_token_logprob_fwd(rows, C.byref(_lib.TokenTargets(t.data_ptr(), 8, 0, 0)), lp.data_ptr(), None, y.data_ptr(), st))
        wg, spread = grad64(p, t, kept, torch.ones_like(d).double())
        check_grad(y, wg, 2 * spread)


@both
@pytest.mark.parametrize("V", [37, 1000])
def test_many_short_rows_some_left_out(cuda_device, dtype, V):
    """More rows than the chip has warps for, so that each takes several; what the left-out ones hold does not count."""
    x, t, g = make(cuda_device, 4, 4001, V, dtype, 29, keep=0.4)
    t[1, :2000] = -1
    t[2, 7] = V
    logp, _, p, kept = rows64(x, t)
    kept[2, 7] = False
    A = torch.randn(4, 4001, device=cuda_device, generator=g)
    wg, spread = grad64(p, torch.where(kept, t, torch.zeros_like(t)), kept, -A.double() / (int(kept.sum()) + 1))
    x[~kept] = math.nan
    out = F.policy_loss(x, t, A, ignore_index=IGN, return_grad=True)
    assert out.grad[2, 7].isnan().all() and out.log_probs.isnan().sum() == 1 and out.loss.isnan()
    out.grad[2, 7], out.log_probs[2, 7], logp[2, 7] = 0, 0, 0
    check_logp(out.log_probs, logp)
    check_grad(out.grad, wg, 2 * spread)


@both
@pytest.mark.parametrize("V", [100, 5000, 50257, 700001])
def test_divergence_of_forbidden_tokens(cuda_device, dtype, V):
    """The policy forbids a token (-inf) that the reference allows: the divergence is infinite, and seen in the loss where it has a weight."""
    x, t, g = make(cuda_device, 2, 2, V, dtype, 30, keep=1.0)
    x[0, 1, int(t[0, 1])] = -math.inf
    A, old = torch.ones(2, device=cuda_device), torch.full((2, 2), -2.0, device=cuda_device)
    for grad in (False, True):
        out = F.policy_loss(x, t, A, old, old, return_grad=grad)
        assert out.kl == math.inf and out.loss.isfinite()
        assert F.policy_loss(x, t, A, old, old, kl_coef=0.1, return_grad=grad).loss == math.inf
        nan = old.clone()
        nan[1, 0] = math.nan
        assert F.policy_loss(x, t, A, old, nan, return_grad=grad).kl.isnan()
    assert (out.grad[0, 1] == 0).all() and out.grad.isfinite().all()   # a ratio of 0


@both
@pytest.mark.parametrize("V", [50, 5001, 50257, 700001])
@pytest.mark.parametrize("T", [0.5, 1.0, 2.0])
def test_distillation_of_forbidden_tokens(cuda_device, dtype, V, T):
    """The student forbids what the teacher likes best or second best: a large or infinite loss, and a gradient of ordinary size."""
    K = 6
    g = torch.Generator(device=cuda_device).manual_seed(31)
    low = torch.finfo(dtype).min
    masks = [-1e4, -1e9, low, -math.inf]
    R = 2 * len(masks) + 2
    x = (torch.randn(1, R, V, device=cuda_device, generator=g) * 2).to(dtype)
    ids = torch.stack([torch.randperm(V, device=cuda_device, generator=g)[:K] for _ in range(R)]).view(1, R, K)
    tl = torch.randn(1, R, K, device=cuda_device, generator=g)
    tl[..., 0], tl[..., 1] = 4.0, 3.5
    for i, v in enumerate(masks + masks):
        x[0, i, ids[0, i, i // len(masks)]] = v
    x[0, R - 2] = 3e38
    x[0, R - 1] = low
    q = torch.softmax(tl.double() / T, -1)
    z = (x.double() - x.double().amax(-1, keepdim=True)) / T
    logp = z - z.exp().sum(-1, keepdim=True).log()
    p = logp.exp()
    _, grad = F.distillation_loss(x, ids, tl, temperature=T, return_grad=True)
    check_grad(grad, p.scatter_add(-1, ids, -q) * T / R, p.scatter_add(-1, ids, q) * T / R)
    want = (q * (q.log() - logp.gather(-1, ids))).sum(-1)[0] * T * T
    for i in range(R):
        for with_grad in (False, True):
            out = F.distillation_loss(x[:, i:i + 1], ids[:, i:i + 1], tl[:, i:i + 1], temperature=T, return_grad=with_grad)
            v, w = float(out[0] if with_grad else out), float(want[i])
            # terms of size |log q| + loss, each to 3e-5; where y = x / T or the loss, before T^2 or after it, is no float32 any more, the
            # loss may be infinite
            near = abs(v - w) <= 3e-5 * (T * T * 20 + w)
            held = max(w, w / (T * T), float(x[0, i].abs().max()) / T) < torch.finfo(F32).max * (1 - 1e-4)
            assert near or (v == math.inf and not held), (i, v, w)


@both
@pytest.mark.parametrize("V", [37, 300, 2051, 50257])
def test_gradients_at_every_alignment(cuda_device, dtype, V):
    """Gradients that begin anywhere relative to 16 bytes, while the logits begin on or beside such a boundary, on another stream than
    the one that made the inputs."""
    B, S, K = 2, 3, 5
    x0, t, g = make(cuda_device, B, S, V, dtype, 25)
    ids, tl = teacher(cuda_device, g, B, S, V, K, dtype)
    n, lib = B * S * V, _lib.load()
    A = torch.randn(B, S, device=cuda_device, generator=g)
    logp64, _, p, kept = rows64(x0, t)
    w = kept.double() / kept.sum().clamp_min(1)
    by_target, spread = grad64(p, t, kept, A.double())
    by_policy = -by_target / kept.sum().clamp_min(1)   # r = 1 without old log-probabilities
    q = torch.softmax(tl.double(), -1)
    by_teacher = p.scatter_add(-1, ids, -q) / (B * S)
    parts = p.scatter_add(-1, ids, q) / (B * S)
    stream = torch.cuda.Stream()
    for lo in (0, 1):
        flat = torch.empty(n + 1, dtype=dtype, device=cuda_device)
        x = flat[lo:lo + n].view(B, S, V)
        x.copy_(x0)
        rows = C.byref(_lib.TokenLogits(x.data_ptr(), B, S, V, S * V, V, 1.0, int(dtype == BF)))
        tt = C.byref(_lib.TokenTargets(t.data_ptr(), 8, 1, IGN))
        pol = C.byref(_lib.PolicyTerms(A.data_ptr(), 1, None, None, 0.2, 0.2, 0.0, 0))
        top = C.byref(_lib.TeacherTop(ids.data_ptr(), tl.data_ptr(), K, 8, int(dtype == BF)))
        torch.cuda.synchronize()
        for off in range(8):
            with torch.cuda.stream(stream):
                st = stream.cuda_stream
                ws = torch.empty(lib.mcb_token_loss_workspace_bytes(B, S), dtype=torch.uint8, device=cuda_device)
                logp, lse, out = (torch.empty(B, S, device=cuda_device) for _ in range(3))
                bufs = [torch.full((n + 40,), 7.0, dtype=dtype, device=cuda_device) for _ in range(3)]
                at = [b[16 + off:].data_ptr() for b in bufs]
                _lib.check(lib.mcb_token_logprob_fwd(rows, tt, logp.data_ptr(), lse.data_ptr(), None, st))
                _lib.check(lib.mcb_token_logprob_bwd(rows, tt, logp.data_ptr(), lse.data_ptr(), A.data_ptr(), 1, at[0], st))
                _lib.check(lib.mcb_policy_loss(rows, tt, pol, 0, logp.data_ptr(), out.data_ptr(), at[1], ws.data_ptr(), ws.numel(), st))
                _lib.check(lib.mcb_distill_loss(rows, top, None, out.data_ptr(), at[2], ws.data_ptr(), ws.numel(), st))
            stream.synchronize()
            check_logp(logp, logp64)
            for b, want, size in zip(bufs, (by_target, by_policy, by_teacher), (spread, spread * w.max(), parts)):
                check_grad(b[16 + off:16 + off + n].view(B, S, V), want, 2 * size)
                assert (b[:16 + off] == 7).all() and (b[16 + off + n:] == 7).all()


@both
@pytest.mark.parametrize("eps,average", [(0.0, False), (0.2, True)])
def test_preference_loss_alone(cuda_device, dtype, eps, average):
    """Without a gradient: the same loss and log-probabilities, bit for bit."""
    for B, S, V in ((2, 3, 50), (6, 5, 8193), (4, 7, 50257)):
        x, t, g = make(cuda_device, B, S, V, dtype, 26)
        ref = torch.randn(B, device=cuda_device, generator=g)
        opts = dict(beta=0.3, label_smoothing=eps, average_log_probs=average, ignore_index=IGN)
        a, b = F.preference_loss(x, t, ref, **opts), F.preference_loss(x, t, ref, return_grad=True, **opts)
        assert a.grad is None and torch.equal(a.loss, b.loss) and torch.equal(a.log_probs, b.log_probs)


LONGEST = {BF: 655353, F32: 655357}   # columns of the longest row that the one-pass kernel takes


@both
@pytest.mark.parametrize("more", [0, 1])
@pytest.mark.parametrize("lo", [0, 1])
def test_longest_rows_of_one_pass(cuda_device, dtype, more, lo):
    """Both sides of the border between the one-pass kernel and the one with three sweeps, from a 16-byte boundary and beside it; rows of
    an odd length, so that each begins elsewhere."""
    V, B, S = LONGEST[dtype] + more, 1, 4
    x0, t, g = make(cuda_device, B, S, V, dtype, 27, keep=1.0)
    flat = torch.empty(B * S * V + 1, dtype=dtype, device=cuda_device)
    x = flat[lo:lo + B * S * V].view(B, S, V)
    x.copy_(x0)
    logp, _, p, kept = rows64(x, t)
    A = torch.randn(B, S, device=cuda_device, generator=g)
    out = F.policy_loss(x, t, A, return_grad=True)
    check_logp(out.log_probs, logp)
    wg, spread = grad64(p, t, kept, -A.double() / S)
    check_grad(out.grad, wg, 2 * spread)
    ids, tl = teacher(cuda_device, g, B, S, V, 9, dtype)
    ids[0, :, 0], ids[0, :, 1] = 0, V - 1
    ids[0, :, 2:] = 1 + ids[0, :, 2:] % (V - 2)
    loss, grad = F.distillation_loss(x, ids, tl, return_grad=True)
    q = torch.softmax(tl.double(), -1)
    check_grad(grad, p.scatter_add(-1, ids, -q) / S, p.scatter_add(-1, ids, q) / S)
    want = (q * (q.log() - p.gather(-1, ids).log())).sum(-1).mean()
    assert abs(float(loss) - float(want)) <= 3e-5 * (1 + abs(float(want)) + float((q * q.log().abs()).sum(-1).mean()))
    assert _lib.device_status() == 0
