"""Masked attention where values are not finite, over long documents: rows that are taken again by themselves."""
import math

import pytest
import torch

from metal_candle_b200 import _lib, backend
from tests.support import packed_reference as ref
from tests.test_gpu_masked_attention import inputs, run

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def fastest(call, times=5):
    """Shortest of some passes after one, in ms."""
    call()
    best = math.inf
    for _ in range(times):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_are_nan_by_right_are_left_at_once(cuda_device, dtype):
    """A diverged run, NaN everywhere: a row is done when its first key has shown it.  (A row that walks over its keys one after the other
    all the same takes hundreds of times as long as a finite pass.)"""
    S, G, d = (16384 if dtype == BF16 else 4096), 2, 64
    q, k, v, dout = inputs(cuda_device, 1, S, 1, G, d, dtype, False, 3)
    mask = backend.attention_mask(batch=1, seq=S, device=cuda_device)
    finite = fastest(lambda: run(q, k, v, dout, G, 0.125, mask, 0.0, None, False))
    for t in (q, k, v, dout):
        t.fill_(math.nan)
    got = run(q, k, v, dout, G, 0.125, mask, 0.0, None, False)
    for name, t in got.items():
        assert torch.isnan(t).all(), name
    took = fastest(lambda: run(q, k, v, dout, G, 0.125, mask, 0.0, None, False))
    assert took <= 4 * finite + 1, (took, finite)


def document_64(q, k, v, dout, scale, dtype):
    """{name: (value, bound)} of one causal document and head, [n, d] each, in float64 on the GPU, a piece of the queries at a time.  Formulas and
    bounds: tests/support/packed_reference.py, for the tensor cores."""
    n, d = q.shape
    u = up = torch.finfo(dtype).eps / 2
    w = 2.0 ** -22
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    out = {name: (torch.zeros(n, d, dtype=torch.float64, device=q.device), torch.zeros(n, d, dtype=torch.float64, device=q.device))
           for name in ("o", "dq", "dk", "dv")}
    out["lse"] = tuple(torch.zeros(n, dtype=torch.float64, device=q.device) for _ in range(2))
    step = 512
    for a in range(0, n, step):
        e = min(n, a + step)
        qc, go, kc, vc = q[a:e], dout[a:e], k[:e], v[:e]
        unseen = torch.arange(e, device=q.device)[None, :] > torch.arange(a, e, device=q.device)[:, None]
        s = (qc @ kc.T).mul_(scale).masked_fill_(unseen, -math.inf)
        z = torch.logsumexp(s, 1)
        p = torch.exp(s - z[:, None])
        top = s.masked_fill_(unseen, 0.0).abs_().amax(1)
        dots = (qc.abs() @ kc.abs().T).mul_(scale).masked_fill_(unseen, 0.0).amax(1)
        ds = (d + 4) * w * dots + 2.0 ** -21 * top.clamp_min(1.0)
        pe = 2 * ds + up + e * w
        o = p @ vc
        eo = pe[:, None] * (p @ vc.abs()) + u * o.abs()
        delta = (go * o).sum(1)
        ddelta = ((u + d * w) * go.abs() * o.abs()).sum(1) + (go.abs() * eo).sum(1)
        grad = (go @ vc.T).sub_(delta[:, None]).mul_(p)
        ge = grad.abs().mul_(pe[:, None]).add_((go.abs() @ vc.abs().T).mul_(d * w).add_(ddelta[:, None]).mul_(p))
        dq = grad @ kc * scale
        for name, value, bound in (("o", o, eo), ("lse", z, ds + e * w + 2.0 ** -21 * z.abs()), ("dq", dq, ge @ kc.abs() * scale + u * dq.abs())):
            out[name][0][a:e], out[name][1][a:e] = value, bound
        for name, value, bound in (("dk", grad.T @ qc * scale, ge.T @ qc.abs() * scale), ("dv", p.T @ go, (p * pe[:, None]).T @ go.abs())):
            out[name][0][:e] += value
            out[name][1][:e] += bound
    for name in ("dk", "dv"):
        out[name][1].add_(u * out[name][0].abs())
    return out


def check(got, want, name):
    value, bound = want
    got = got.double()
    assert torch.isfinite(got).all(), name
    off = float(((got - value).abs() - bound).max())
    assert off <= 1e-30, f"{name}: {off:.3g} over its bound"


def test_a_long_document_behind_one_that_is_not_finite(cuda_device):
    """131109 positions, of which the first ten are NaN and another document's: the long one's first block of keys holds them, so that every one of its
    rows comes out NaN at first (0 x NaN) and is taken again from up to 131099 keys.  However long that is, no wait may run out meanwhile."""
    S, d, first = 131109, 64, 10
    q, k, v, dout = inputs(cuda_device, 1, S, 1, 1, d, BF16, False, 5)
    for t in (q, k, v, dout):
        t[:, :first] = math.nan
    ids = torch.ones(1, S, dtype=torch.int32, device=cuda_device)
    ids[:, :first] = 0
    assert _lib.device_status() == 0
    got = run(q, k, v, dout, 1, 0.125, backend.attention_mask(ids), 0.0, None, False)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    want = document_64(*(t[0, first:] for t in (q, k, v, dout)), 0.125, BF16)
    for name, value in want.items():
        check(got[name][0, first:], value, name)
        assert torch.isnan(got[name][0, :first]).all(), name


def test_a_nan_late_in_a_long_document(cuda_device):
    """One NaN key at position 100000 of 131072: the queries before it are what they are without it, those from it on are NaN, each behind a walk over all
    keys before that one, and so is every key's gradient."""
    S, d, at = 131072, 64, 100000
    q, k, v, dout = inputs(cuda_device, 1, S, 1, 1, d, BF16, False, 6)
    mask = backend.attention_mask(batch=1, seq=S, device=cuda_device)
    clean = run(q, k, v, dout, 1, 0.125, mask, 0.0, None, False)
    k[0, at, 7] = math.nan
    assert _lib.device_status() == 0
    got = run(q, k, v, dout, 1, 0.125, mask, 0.0, None, False)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    tile = at // 128 * 128
    for name in ("o", "lse", "dq"):
        assert torch.equal(got[name][0, :tile], clean[name][0, :tile]), name
        assert torch.isfinite(got[name][0, tile:at]).all() and torch.isnan(got[name][0, at:]).all(), name
    for name in ("dk", "dv"):
        assert torch.isnan(got[name][0, :at + 1]).all(), name


def test_many_rows_taken_again(cuda_device):
    """More items than the CTAs that run at once, most of them with rows to take again, of every quadrant: each is done, once.  Documents of 100
    positions, every third NaN."""
    B, S, G, d, doc = 40, 4000, 3, 64, 100
    q, k, v, dout = inputs(cuda_device, B, S, 1, G, d, BF16, True, 7)
    number = torch.arange(S, device=cuda_device) // doc
    ids = (number % 7).to(torch.int32).expand(B, S).contiguous()
    mask = backend.attention_mask(ids)
    dirty = number % 3 == 1
    q.view(B, G, S, d)[:, :, dirty] = math.nan
    k[:, dirty] = v[:, dirty] = math.nan
    dout.view(B, S, G * d)[:, dirty] = math.nan
    got = run(q, k, v, dout, G, 0.125, mask, 0.0, None, True)
    again = run(q, k, v, dout, G, 0.125, mask, 0.0, None, True)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    rows = lambda t: t.view(B, G, S, -1).transpose(1, 2) if t.shape[:2] == (B, G * S) else t.view(B, S, -1)  # noqa: E731
    for name in got:
        a, b = rows(got[name]), rows(again[name])
        assert torch.isnan(a[:, dirty]).all(), name
        assert torch.isfinite(a[:, ~dirty]).all() and torch.equal(a[:, ~dirty], b[:, ~dirty]), name
    for b in (0, 23, B - 1):
        for at in range(0, S, doc):
            if dirty[at]:
                continue
            part = lambda t: t.view(B, -1, S, t.shape[-1])[b, :, at:at + doc].reshape(1, -1, t.shape[-1])  # noqa: E731
            token = lambda t: t.view(B, S, G * d)[b, at:at + doc]  # noqa: E731
            want = ref.attention(part(q), part(k), part(v), token(dout), [[0] * doc], None, G, 0.125, 0.0, None, True, BF16, True)
            for name, value in want.items():
                x = token(got[name]) if name == "o" else part(got[name][..., None]).view(1, -1) if name == "lse" else part(got[name])
                ref.check(x, value, f"{name} of {b}, {at}")


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F32, 8)])
def test_scores_near_the_lowest_number(cuda_device, dtype, d):
    """Scores of -2.25e38, -3.25e38 in units of log 2, are scores: a row that has no others takes the mean of its keys."""
    S = 70
    q, k, v, _ = inputs(cuda_device, 1, S, 1, 1, d, dtype, False, 8)
    q.zero_()
    k.zero_()
    q[..., 0], k[..., 0] = 1.5e19, -1.5e19
    o, lse = backend.attention_masked_forward(q, k, v, 1, 1.0, backend.attention_mask(batch=1, seq=S, device=cuda_device))
    score = float(q[0, 0, 0].double() * k[0, 0, 0].double())
    assert ((lse.double() - score).abs() <= 2.0 ** -21 * abs(score)).all()
    for i in range(S):   # all scores equal: weights of 1, summed and divided in float32, the result rounded
        want = v[0, :i + 1].double().mean(0)
        bound = (torch.finfo(dtype).eps / 2 + (S + 2) * 2.0 ** -22) * v[0, :i + 1].double().abs().mean(0)
        assert ((o[0, i].double() - want).abs() <= bound).all(), i


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_late_nan_takes_no_walk_over_the_keys_before_it(cuda_device, dtype):
    """A query from the NaN key on has weights whose sum is NaN, and a key before it a query whose log-sum-exp is: NaN by right, which shows without taking
    the row again.  (What is left are the rows of one tile before the key.)"""
    S, G, d = (16384 if dtype == BF16 else 4096), 2, 64
    at = S // 2 + 1   # a tile's second position
    q, k, v, dout = inputs(cuda_device, 1, S, 1, G, d, dtype, False, 3)
    mask = backend.attention_mask(batch=1, seq=S, device=cuda_device)
    finite = fastest(lambda: run(q, k, v, dout, G, 0.125, mask, 0.0, None, False))
    k[0, at, 3] = math.nan
    got = run(q, k, v, dout, G, 0.125, mask, 0.0, None, False)
    for name in ("o", "lse", "dq"):
        t = got[name].view(G, S, -1)
        assert torch.isfinite(t[:, :at]).all() and torch.isnan(t[:, at:]).all(), name
    assert torch.isnan(got["dk"]).all() and torch.isnan(got["dv"]).all()
    took = fastest(lambda: run(q, k, v, dout, G, 0.125, mask, 0.0, None, False))
    # one row a head, of half the sequence, by one warp: 256 (64) steps of some microseconds, three times
    assert took <= 4 * finite + 6, (took, finite)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_taken_again_on_two_streams_and_in_a_graph(cuda_device, dtype):
    """The same bits whatever runs beside them, eager, on two streams at a time, and replayed; and finite passes between them."""
    B, S, G, d = 3, 1500, 4, 64
    ids = (torch.arange(S, device=cuda_device) // 170).to(torch.int32).expand(B, S).contiguous()
    mask = backend.attention_mask(ids)
    clean = inputs(cuda_device, B, S, 1, G, d, dtype, True, 4)
    dirty = [t.clone() for t in clean]
    odd = ids[0] % 2 == 1
    dirty[0].view(B, G, S, d)[:, :, odd] = math.nan
    dirty[1][:, odd] = dirty[2][:, odd] = math.inf
    step = lambda t: run(*t, G, 0.125, mask, 15.0, None, True)  # noqa: E731
    bits = lambda out: {n: t.view(torch.int16 if t.dtype == BF16 else torch.int32).clone() for n, t in out.items()}  # noqa: E731
    want = [bits(step(t)) for t in (clean, dirty)]
    assert all(torch.isfinite(t.view(dtype if n != "lse" else F32)).all() for n, t in want[0].items())
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((step(dirty if i % 4 < 2 else clean), i % 4 < 2))
    torch.cuda.synchronize()
    for out, bad in outs:
        assert all(torch.equal(x, want[bad][n]) for n, x in bits(out).items())
    buf = [t.clone() for t in clean]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(buf)
    for bad in (1, 0, 1):
        for b, t in zip(buf, (clean, dirty)[bad]):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, want[bad][n]) for n, x in bits(held).items())
    assert _lib.device_status() == 0
