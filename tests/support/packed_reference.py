"""Attention under document / prefix masks in float64 on the CPU, with the gradients' formulas written out and, beside every output, how
far a float32 or bfloat16 kernel may be from it.

The bounds count roundings.  u is half a step of the storage type, w half a step of a float32 sum (2^-24; 2^-22 for the tensor
cores, whose sums align their terms).  With A = |q| |k|^T scale and n terms to a sum:
  scores        ds = (d + 4) w A + 2^-21 max(|s|, 1)           (the dot; scale, exponent and log-sum-exp in base 2, cap, bias)
  P             2 ds P + u P where it is rounded for the tensor cores
  o             (2 ds + u_p + n w) (P |v|) + u |o|
  delta         u |do| |o| + d w |do| |o|                      (o is read back rounded)
  dS            (2 ds + u_p) |dS| + P (d w |do| |v| + d delta) + P |dP - delta| (2 ds / cap + 2^-21) where there is a cap
  dq, dk, dv    the sums of these against |k|, |q|, |do|, and u of the result
"""
import math

import torch


def runs(ids):
    """(first, behind last) of every run of equal ids that are not negative."""
    out, at = [], 0
    while at < len(ids):
        end = at + 1
        while end < len(ids) and ids[end] == ids[at]:
            end += 1
        if ids[at] >= 0:
            out.append((at, end))
        at = end
    return out


def visible(ids, prefix):
    """[S, S] bool: query i sees key j."""
    S = len(ids)
    see = torch.zeros(S, S, dtype=torch.bool)
    for a, e in runs(ids):
        lead = a
        while prefix is not None and lead < e and prefix[lead]:
            lead += 1
        i = torch.arange(a, e)
        see[a:e, a:e] = (i[None, :] <= i[:, None]) | (i[None, :] < lead)
    return see


def attention(q, k, v, dout, ids, prefix, groups, scale, softcap, slopes, token_major, dtype, tensor_cores):
    """{name: (value, bound)} for o, lse and, with dout, dq, dk, dv; laid out as the kernels do.  ids, prefix: lists per sequence."""
    u = torch.finfo(dtype).eps / 2
    up = u if tensor_cores else 0.0
    w = 2.0 ** -22 if tensor_cores else 2.0 ** -24
    nb, S, d = k.shape
    B = len(ids)
    Hk = nb // B
    f64 = torch.float64
    q, k, v = (t.detach().cpu().to(f64) for t in (q, k, v))
    q = q.view(nb, groups, S, d)
    if dout is not None:
        dout = dout.detach().cpu().to(f64)
        dout = dout.view(B, S, Hk, groups, d).permute(0, 2, 3, 1, 4).reshape(nb, groups, S, d) if token_major else dout.view(nb, groups, S, d)
    zeros = lambda *s: torch.zeros(*s, dtype=f64)  # noqa: E731
    o, eo = zeros(nb, groups, S, d), zeros(nb, groups, S, d)
    lse, el = zeros(nb, groups, S), zeros(nb, groups, S)
    dq, eq = zeros(nb, groups, S, d), zeros(nb, groups, S, d)
    dk, ek, dv, ev = (zeros(nb, S, d) for _ in range(4))
    at = torch.arange(S, dtype=f64)
    far = (at[:, None] - at[None, :]).abs()
    for n in range(nb):
        b, hk = divmod(n, Hk)
        see = visible(ids[b], None if prefix is None else prefix[b])
        some = see.any(1)
        # masked positions' values count for nothing, whatever they are
        used_q, used_k = some[:, None], see.any(0)[:, None]
        kn, vn = (torch.where(used_k, t[n], torch.zeros((), dtype=f64)) for t in (k, v))
        for g in range(groups):
            qn = torch.where(used_q, q[n, g], torch.zeros((), dtype=f64))
            raw = qn @ kn.T * scale
            bent = torch.tanh(raw / softcap) if softcap > 0 else None
            s = softcap * bent if softcap > 0 else raw
            if slopes is not None:
                s = s - float(slopes[hk * groups + g]) * far
            s = s.masked_fill(~see, -math.inf)
            z = torch.logsumexp(s, -1)
            p = torch.where(see, torch.exp(s - torch.where(some, z, torch.zeros((), dtype=f64))[:, None]), torch.zeros((), dtype=f64))
            size = torch.where(see, s.abs(), torch.zeros((), dtype=f64))
            ds = (d + 4) * w * (qn.abs() @ kn.abs().T) * abs(scale) + 2.0 ** -21 * size.clamp_min(1.0).amax(1, keepdim=True)
            ds = torch.where(see, ds, torch.zeros((), dtype=f64)).amax(1, keepdim=True).expand(S, S)
            pe = (2 * ds + up + S * w) * p
            o[n, g], eo[n, g] = p @ vn, pe @ vn.abs()
            eo[n, g] += u * o[n, g].abs()
            lse[n, g], el[n, g] = z, ds[:, 0] + S * w + 2.0 ** -21 * torch.where(some, z, torch.zeros((), dtype=f64)).abs()
            if dout is None:
                continue
            do = torch.where(used_q, dout[n, g], torch.zeros((), dtype=f64))
            delta = (do * o[n, g]).sum(-1, keepdim=True)
            ddelta = ((u + d * w) * do.abs() * o[n, g].abs()).sum(-1, keepdim=True) + (do.abs() * eo[n, g]).sum(-1, keepdim=True)
            dp = do @ vn.T
            slope = 1 - bent * bent if softcap > 0 else torch.ones_like(p)
            grad = p * (dp - delta) * slope
            ge = (2 * ds + up + S * w) * grad.abs() + p * (d * w * (do.abs() @ vn.abs().T) + ddelta)
            if softcap > 0:
                ge = ge + p * (dp - delta).abs() * (2 * ds / softcap + 2.0 ** -21)
            dv[n] += p.T @ do
            ev[n] += pe.T @ do.abs()
            dq[n, g], eq[n, g] = grad @ kn * scale, ge @ kn.abs() * abs(scale)
            dk[n] += grad.T @ qn * scale
            ek[n] += ge.T @ qn.abs() * abs(scale)
    eq, ek, ev = eq + u * dq.abs(), ek + u * dk.abs(), ev + u * dv.abs()
    major = (lambda t: t.view(B, Hk, groups, S, d).permute(0, 3, 1, 2, 4).reshape(B * S, Hk * groups * d)) if token_major else (lambda t: t.reshape(nb, groups * S, d))  # noqa: E731
    out = {"o": (major(o), major(eo)), "lse": (lse.view(nb, groups * S), el.view(nb, groups * S))}
    if dout is not None:
        out.update(dq=(dq.view(nb, groups * S, d), eq.view(nb, groups * S, d)), dk=(dk, ek), dv=(dv, ev))
    return out


def check(got, want, name):
    """got within its bound of want = (value, bound) everywhere, and infinite where it is."""
    value, bound = want
    got = got.detach().cpu().to(torch.float64)
    assert got.shape == value.shape, (name, got.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(got[~fine], value[~fine]), f"{name}: values that are not finite"
    off = (got - value).abs()[fine] - bound[fine]
    assert torch.isfinite(got[fine]).all(), f"{name}: {int((~torch.isfinite(got[fine])).sum())} values are not finite"
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1e-30, f"{name}: {worst:.3g} over its bound ({int((off > 0).sum())} of {off.numel()} values)"
