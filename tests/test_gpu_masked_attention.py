"""Attention under document / prefix masks, capped scores and distance bias against the formulas in float64 (tests/support/packed_reference.py,
where the bounds are derived)."""
import math
import random

import pytest
import torch

from metal_candle_b200 import backend
from tests.support import packed_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def make_ids(kind, B, S, seed):
    """Document ids and prefix marks per sequence, as lists."""
    rng = random.Random(seed)
    ids, prefix = [], []
    for b in range(B):
        row, marks = [], []
        if kind == "one":
            row, marks = [0] * S, [False] * S
        elif kind == "padding":
            row, marks = [-1] * S, [True] * S
        else:
            doc = 0
            while len(row) < S:
                n = min(S - len(row), max(1, int(rng.lognormvariate(math.log(max(2, S / 4)), 1.0))))
                pad = rng.random() < 0.25
                lead = rng.randint(0, n) if kind == "prefix" else 0
                # ids in no order, the same one again after another; padding of several values
                row += [rng.choice([-1, -7]) if pad else [5, 0, 3][doc % 3]] * n
                marks += [i < lead or (i > lead and rng.random() < 0.3) for i in range(n)]
                doc += 1
        ids.append(row)
        prefix.append(marks)
    return ids, prefix if kind in ("prefix", "padding") else None


def inputs(dev, B, S, Hk, G, d, dtype, token_major, seed, spread=2.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
    q, k, v = (rand(B * Hk, G * S, d) * spread).to(dtype), rand(B * Hk, S, d).to(dtype), rand(B * Hk, S, d).to(dtype)
    dout = (rand(B * S, Hk * G * d) if token_major else rand(B * Hk, G * S, d)).to(dtype)
    return q, k, v, dout


def run(q, k, v, dout, groups, scale, mask, softcap, slopes, token_major):
    how = dict(groups=groups, scale=scale, mask=mask, softcap=softcap, slopes=slopes, token_major=token_major)
    o, lse = backend.attention_masked_forward(q, k, v, **how)
    dq, dk, dv = backend.attention_masked_backward(q, k, v, o, lse, dout, **how)
    return dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)


def mask_of(dev, ids, prefix, dtype=torch.int32):
    return backend.attention_mask(torch.tensor(ids, dtype=dtype, device=dev), None if prefix is None else torch.tensor(prefix, device=dev))


CASES = [
    # B, S, Hk, G, d, dtype, documents, softcap, bias, token_major
    (1, 1, 1, 1, 64, BF16, "one", 0.0, False, False),
    (1, 2, 1, 3, 64, BF16, "docs", 0.0, False, True),
    (2, 63, 2, 1, 64, BF16, "docs", 0.0, False, False),
    (2, 64, 1, 2, 64, BF16, "prefix", 0.0, False, True),
    (1, 65, 2, 7, 64, BF16, "docs", 30.0, False, True),
    (3, 127, 1, 1, 64, BF16, "prefix", 5.0, True, False),
    (1, 128, 2, 2, 64, BF16, "one", 0.0, True, True),
    (2, 129, 2, 2, 64, BF16, "docs", 0.0, True, False),
    (1, 300, 2, 7, 64, BF16, "prefix", 0.0, False, True),
    (2, 515, 1, 4, 64, BF16, "docs", 50.0, True, True),
    (1, 1100, 1, 2, 64, BF16, "prefix", 0.0, False, False),
    (2, 640, 2, 1, 64, BF16, "padding", 0.0, False, True),
    (1, 1, 2, 1, 64, F32, "one", 0.0, False, True),
    (2, 19, 2, 3, 64, F32, "prefix", 20.0, True, False),
    (1, 64, 1, 2, 32, F32, "docs", 0.0, False, True),
    (2, 130, 1, 2, 80, F32, "docs", 0.0, True, True),
    (1, 333, 2, 1, 128, F32, "prefix", 8.0, False, False),
    (2, 200, 1, 3, 8, F32, "docs", 0.0, True, False),
    (1, 96, 1, 1, 64, F32, "padding", 0.0, False, False),
    (1, 193, 2, 2, 128, BF16, "prefix", 30.0, True, True),
    (2, 70, 1, 2, 40, BF16, "docs", 0.0, False, False),
]


@pytest.mark.parametrize("B,S,Hk,G,d,dtype,kind,softcap,bias,token_major", CASES)
def test_against_the_formulas(cuda_device, B, S, Hk, G, d, dtype, kind, softcap, bias, token_major):
    ids, prefix = make_ids(kind, B, S, S)
    mask = mask_of(cuda_device, ids, prefix, torch.int64 if S % 2 else torch.int32)
    q, k, v, dout = inputs(cuda_device, B, S, Hk, G, d, dtype, token_major, S + d, 6.0 if softcap else 2.0)
    slopes = 2.0 ** -torch.arange(1, Hk * G + 1, device=cuda_device, dtype=F32) if bias else None
    scale = 1.0 / math.sqrt(d)
    got = run(q, k, v, dout, G, scale, mask, softcap, slopes, token_major)
    want = ref.attention(q, k, v, dout, ids, prefix, G, scale, softcap, slopes, token_major, dtype, dtype == BF16 and d == 64)
    for name, value in want.items():
        ref.check(got[name], value, name)
    again = run(q, k, v, dout, G, scale, mask, softcap, slopes, token_major)
    for name in got:
        assert torch.equal(got[name], again[name]), f"{name}: other bits the second time"


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F32, 64), (F32, 32)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_does_not_matter(cuda_device, dtype, d, bad):
    """Padding and a neighbouring document full of NaN or infinities leave the other documents as they are."""
    B, S, Hk, G, scale = 2, 200, 2, 2, 0.125
    ids = [[0] * 50 + [-1] * 20 + [1] * 70 + [2] * 60, [-1] * 3 + [4] * 40 + [5] * 157]
    dirty = [(0, 50, 70), (0, 140, 200), (1, 0, 3), (1, 43, 200)]   # padding, and whole documents
    for token_major in (False, True):
        q, k, v, dout = inputs(cuda_device, B, S, Hk, G, d, dtype, token_major, 5)
        mask = mask_of(cuda_device, ids, None)
        want = ref.attention(q, k, v, dout, ids, None, G, scale, 10.0, None, token_major, dtype, dtype == BF16)
        clean = torch.ones(B, S, dtype=torch.bool)
        for b, a, e in dirty:
            clean[b, a:e] = False
            q.view(B, Hk, G, S, d)[b, :, :, a:e] = bad
            k.view(B, Hk, S, d)[b, :, a:e] = bad
            v.view(B, Hk, S, d)[b, :, a:e] = bad
            (dout.view(B, S, Hk, G, d)[b, a:e] if token_major else dout.view(B, Hk, G, S, d)[b, :, :, a:e]).fill_(bad)
        got = run(q, k, v, dout, G, scale, mask, 10.0, None, token_major)
        rows = dict(lse=clean[:, None, None, :].expand(B, Hk, G, S), dq=clean[:, None, None, :, None].expand(B, Hk, G, S, d),
                    dk=clean[:, None, :, None].expand(B, Hk, S, d), dv=clean[:, None, :, None].expand(B, Hk, S, d))
        rows["o"] = clean[:, :, None].expand(B, S, Hk * G * d) if token_major else rows["dq"]
        for name, keep in rows.items():
            value, bound = want[name]
            keep = keep.reshape(value.shape)
            ref.check(got[name].cpu()[keep], (value[keep], bound[keep]), name)
        # padding itself: nothing seen, no gradient
        pad = torch.zeros(B, S, dtype=torch.bool)
        pad[0, 50:70] = pad[1, 0:3] = True
        heads = pad[:, None, None, :].expand(B, Hk, G, S)
        assert (got["lse"].cpu().view(B, Hk, G, S)[heads] == -math.inf).all()
        assert (got["dq"].cpu().view(B, Hk, G, S, d)[heads] == 0).all()
        assert (got["dk"].cpu().view(B, Hk, S, d)[pad[:, None].expand(B, Hk, S)] == 0).all()
        assert (got["dv"].cpu().view(B, Hk, S, d)[pad[:, None].expand(B, Hk, S)] == 0).all()
        o = got["o"].cpu()
        o = o.view(B, S, Hk, G, d).permute(0, 2, 3, 1, 4) if token_major else o.view(B, Hk, G, S, d)
        assert (o[heads] == 0).all()


def expected_intervals(ids, prefix):
    S = len(ids)
    rows, keys = [(i, i) for i in range(S)], [(i, i) for i in range(S)]
    for a, e in ref.runs(ids):
        lead = a
        while prefix is not None and lead < e and prefix[lead]:
            lead += 1
        for i in range(a, e):
            rows[i] = (a, max(i + 1, lead))
            keys[i] = (a if i < lead else i, e)
    return rows, keys


@pytest.mark.parametrize("B,S,longest", [(3, 1, 1), (2, 1000, 3), (1, 32768, 40), (1, 32769, 40000), (2, 70001, 900), (1, 140000, 139000), (1, 100000, 100000)])
def test_the_mask_as_intervals(cuda_device, B, S, longest):
    """The intervals that the kernels read, over more than one word of every bitmap level."""
    rng = random.Random(S)
    ids, prefix = [], []
    for b in range(B):
        row, marks = [], []
        while len(row) < S:
            n = min(S - len(row), rng.randint(max(1, longest // 2), longest))
            lead = rng.choice([0, n, rng.randint(0, n)])
            row += [rng.randint(-1, 3)] * n
            marks += [True] * lead + [False] * (n - lead)
        ids.append(row)
        prefix.append(marks)
    for pre in (None, prefix):
        mask = mask_of(cuda_device, ids, pre, torch.int64)
        words = mask.block.view(torch.int32).cpu()
        n, tiles = B * S, (S + 127) // 128
        rows, keys = words[:2 * n].view(B, S, 2), words[2 * n:4 * n].view(B, S, 2)
        at = 4 * n
        ranges = words[at:at + 4 * B * tiles].view(2, B, tiles, 2)
        at = (at + 4 * B * tiles + 3) // 4 * 4
        work = words[at:at + 8 * B * tiles].view(2, B * tiles, 4)
        for b in range(B):
            want_rows, want_keys = expected_intervals(ids[b], None if pre is None else pre[b])
            for got, want, tile in ((rows[b], want_rows, ranges[0, b]), (keys[b], want_keys, ranges[1, b])):
                want = torch.tensor(want, dtype=torch.int32)
                assert torch.equal(got, want)
                for t in range(tiles):
                    part = want[t * 128:(t + 1) * 128]
                    part = part[part[:, 0] < part[:, 1]]
                    first, count = tile[t].tolist()
                    if len(part) == 0:
                        assert count == 0
                    else:
                        assert first == int(part[:, 0].min()) // 64 and first + count == (int(part[:, 1].max()) + 63) // 64
        for k in range(2):
            order = (work[k, :, 0] * tiles + work[k, :, 1]).long()
            assert sorted(order.tolist()) == list(range(B * tiles))
            assert torch.equal(work[k, :, 2:], ranges[k].reshape(-1, 2)[order])
            for b in range(B):   # the longest tiles of a sequence first, by classes of a thousandth of the longest
                counts = work[k, work[k, :, 0] == b, 3].double()
                assert (counts[:-1] - counts[1:] >= -counts.max() / 1000).all()


def test_whole_sequences_are_the_causal_kernel(cuda_device):
    """No documents, no prefix: what attention_causal_ragged_forward and _backward compute, up to the rounding of either."""
    B, S, Hk, G, d = 2, 333, 2, 7, 64
    q, k, v, dout = inputs(cuda_device, B, S, Hk, G, d, BF16, True, 3)
    mask = backend.attention_mask(batch=B, seq=S, device=cuda_device)
    got = run(q, k, v, dout, G, 0.125, mask, 0.0, None, True)
    want = ref.attention(q, k, v, dout, [[0] * S] * B, None, G, 0.125, 0.0, None, True, BF16, True)
    o, lse = backend.attention_causal_ragged_forward(q, k, v, G, 0.125, kv_heads=Hk)
    dq, dk, dv = backend.attention_causal_ragged_backward(q, k, v, o, lse, dout, G, 0.125, kv_heads=Hk)
    for name, other in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items():
        value, bound = want[name]
        ref.check(got[name], (other.cpu().double(), 2 * bound), name)


def test_gradients_against_differences(cuda_device):
    """float32: the derivative of sum(o * w) along random directions of q, k and v, by central differences of the forward pass."""
    B, S, Hk, G, d, scale, cap = 1, 40, 2, 2, 16, 0.25, 4.0
    ids, prefix = make_ids("prefix", B, S, 11)
    mask = mask_of(cuda_device, ids, prefix)
    q, k, v, dout = inputs(cuda_device, B, S, Hk, G, d, F32, False, 8)
    slopes = torch.tensor([0.1, 0.02, 0.3, 0.0], device=cuda_device)
    got = run(q, k, v, dout, G, scale, mask, cap, slopes, False)
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    eps = 2.0 ** -7
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        way = torch.randn(t.shape, device=cuda_device, generator=gen)
        ends = []
        for sign in (1, -1):
            args = [t + sign * eps * way if t is x else x for x in (q, k, v)]
            o, _ = backend.attention_masked_forward(*args, groups=G, scale=scale, mask=mask, softcap=cap, slopes=slopes)
            ends.append((o.double() * dout.double()).sum())
        difference = float(ends[0] - ends[1]) / (2 * eps)
        slope = float((got[name].double() * way.double()).sum())
        # third derivatives of order 1 a position over eps^2 / 6 of the square of the way's size, and the outputs' rounding over eps
        size = float((got[name].double() * way.double()).abs().sum())
        noise = float(dout.double().abs().sum()) * 2.0 ** -20 / eps
        assert abs(difference - slope) <= 0.02 * size + noise, (name, difference, slope)


def test_streams_graphs_and_two_at_once(cuda_device):
    B, S, Hk, G, d = 2, 257, 2, 2, 64
    ids, prefix = make_ids("prefix", B, S, 4)
    ids_t = torch.tensor(ids, dtype=torch.int32, device=cuda_device)
    pre_t = torch.tensor(prefix, device=cuda_device)
    for dtype in (BF16, F32):
        q, k, v, dout = inputs(cuda_device, B, S, Hk, G, d, dtype, True, 9)
        q2, k2, v2, dout2 = inputs(cuda_device, B, S, Hk, G, d, dtype, True, 10)
        step = lambda *t: run(*t, G, 0.125, backend.attention_mask(ids_t, pre_t), 20.0, None, True)  # noqa: E731
        want, want2 = step(q, k, v, dout), step(q2, k2, v2, dout2)
        torch.cuda.synchronize()
        # two streams at a time
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        outs = []
        for _ in range(3):
            for stream, t in zip(streams, ((q, k, v, dout), (q2, k2, v2, dout2))):
                with torch.cuda.stream(stream):
                    outs.append(step(*t))
        torch.cuda.synchronize()
        for i, got in enumerate(outs):
            for name in got:
                assert torch.equal(got[name], (want2 if i % 2 else want)[name])
        # captured, replayed on other inputs and other documents
        buf = [t.clone() for t in (q, k, v, dout)]
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*buf)
        torch.cuda.current_stream().wait_stream(side)
        with torch.cuda.graph(graph):
            held = step(*buf)
        for other, expect in (((q2, k2, v2, dout2), want2), ((q, k, v, dout), want)):
            for b, t in zip(buf, other):
                b.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            for name in held:
                assert torch.equal(held[name], expect[name])
        old = ids_t.clone()
        ids_t.copy_(torch.full_like(ids_t, 1))
        graph.replay()
        changed = held["o"].clone()
        expect = step(q, k, v, dout)["o"]
        ids_t.copy_(old)
        assert torch.equal(changed, expect) and not torch.equal(changed, want["o"])


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F32, 40)])
def test_values_that_are_not_finite_stay_in_their_document(cuda_device, dtype, d):
    """A NaN query, key, value or output gradient makes its own document's rows NaN as the formulas say and leaves the others what they are.

    Not to the bit: a row of a tile that meets the NaN (0 x NaN in a product) is computed again by itself, and there the weights are not
    rounded to bfloat16 (u_p of the bounds is 0 there), so both results are within the bounds and differ by no more than their sum."""
    B, S, Hk, G = 1, 300, 1, 2
    ids = [[0] * 130 + [1] * 170]
    mask = mask_of(cuda_device, ids, None)
    base = inputs(cuda_device, B, S, Hk, G, d, dtype, False, 12)
    want = ref.attention(*base, ids, None, G, 0.125, 0.0, None, False, dtype, dtype == BF16)
    for which, at in (("q", 40), ("k", 40), ("v", 40), ("dout", 40)):
        q, k, v, dout = (t.clone() for t in base)
        t = dict(q=q, k=k, v=v, dout=dout)[which]
        t[0, at, 3] = math.nan   # head 0 of the first document
        got = run(q, k, v, dout, G, 0.125, mask, 0.0, None, False)
        o, dq = got["o"].view(G, S, d), got["dq"].view(G, S, d)
        nan = {name: torch.isnan(got[name]).view(-1, S, d).any(0).any(-1).cpu() for name in ("o", "dq", "dk", "dv")}
        seen = torch.zeros(S, dtype=torch.bool)
        if which == "q":     # one query row: its o; dq of it; dk and dv of the keys that it sees
            seen[:41] = True
            assert nan["o"].nonzero().flatten().tolist() == [40] and nan["dq"].nonzero().flatten().tolist() == [40]
            assert torch.equal(nan["dk"], seen) and torch.equal(nan["dv"], seen)
        elif which == "k":   # the queries that see it
            seen[40:130] = True
            assert torch.equal(nan["o"], seen) and torch.equal(nan["dq"], seen)
        elif which == "v":
            seen[40:130] = True
            assert torch.equal(nan["o"], seen) and torch.equal(nan["dq"], seen)
            assert torch.isfinite(o[:, :130, :3]).all() and torch.isnan(o[:, 40:130, 3]).all()   # the other columns are what they are
        else:
            seen[:41] = True
            assert not nan["o"].any() and nan["dq"].nonzero().flatten().tolist() == [40]
            assert torch.equal(nan["dk"], seen)
        for name in ("o", "dq", "dk", "dv"):
            ref.check(got[name].view(-1, S, d)[:, 130:], tuple(t.view(-1, S, d)[:, 130:] for t in want[name]), f"{name} with {which}")


def test_one_mask_on_two_streams_and_prefix_alone(cuda_device):
    B, S, Hk, G, d = 2, 900, 2, 3, 64
    prefix = torch.zeros(B, S, dtype=torch.uint8, device=cuda_device)
    prefix[0, :333] = 1
    prefix[1, 5:] = 1   # not leading: counts for nothing
    mask = backend.attention_mask(prefix=prefix)
    a, b = inputs(cuda_device, B, S, Hk, G, d, BF16, True, 1), inputs(cuda_device, B, S, Hk, G, d, BF16, True, 2)
    want = [run(*t, G, 0.125, mask, 0.0, None, True) for t in (a, b)]
    value = ref.attention(*a, [[0] * S] * B, prefix.bool().tolist(), G, 0.125, 0.0, None, True, BF16, True)
    for name, v in value.items():
        ref.check(want[0][name], v, name)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(8):
        for stream, t in zip(streams, (a, b)):
            with torch.cuda.stream(stream):
                got.append(run(*t, G, 0.125, mask, 0.0, None, True))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(out[n], want[i % 2][n]) for n in out)


def test_many_short_items(cuda_device):
    """More items than CTAs by far, most of them of one block, some of none: every one is done once."""
    B, S, Hk, G, d = 600, 40, 2, 2, 64
    rng = random.Random(3)
    ids = [[-1] * S if rng.random() < 0.3 else [i // rng.randint(1, 9) for i in range(S)] for _ in range(B)]
    mask = mask_of(cuda_device, ids, None)
    q, k, v, dout = inputs(cuda_device, B, S, Hk, G, d, BF16, False, 4)
    got = run(q, k, v, dout, G, 0.125, mask, 0.0, None, False)
    want = ref.attention(q, k, v, dout, ids, None, G, 0.125, 0.0, None, False, BF16, True)
    for name, value in want.items():
        ref.check(got[name], value, name)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sequences_beyond_one_launch_of_the_mask(cuda_device, dtype):
    """40000 positions: the mask is made in two launches; documents at the start, across position 32768 and at the end."""
    S, Hk, G, d = 40000, 1, 2, 64
    rng, ids, spans = random.Random(5), [], []
    while len(ids) < S:
        n = min(S - len(ids), rng.randint(1, 400))
        spans.append((len(ids), len(ids) + n))
        ids += [len(spans) % 3] * n
    q, k, v, dout = inputs(cuda_device, 1, S, Hk, G, d, dtype, False, 9)
    got = run(q, k, v, dout, G, 0.125, mask_of(cuda_device, [ids], None), 0.0, None, False)
    for a, e in [spans[0], next(s for s in spans if s[0] <= 32768 < s[1]), spans[-1]]:
        part = lambda t, n: t.view(n, S, -1)[:, a:e].reshape(1, n * (e - a), -1).contiguous()  # noqa: E731
        want = ref.attention(part(q, G), part(k, 1), part(v, 1), part(dout, G), [[0] * (e - a)], None, G, 0.125, 0.0, None, False, dtype, dtype == BF16)
        for name, n in (("o", G), ("dq", G), ("dk", 1), ("dv", 1)):
            ref.check(part(got[name], n), want[name], f"{name} of [{a}, {e})")
        ref.check(got["lse"].view(G, S)[:, a:e].reshape(1, -1), want["lse"], "lse")


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F32, 64), (F32, 40), (BF16, 128)])
@pytest.mark.parametrize("softcap,bias", [(0.0, False), (30.0, True)])
def test_documents_of_one_token(cuda_device, dtype, d, softcap, bias):
    """A softmax over one key does not depend on the score: dq is 0, exactly, and so is dk (on the tensor cores up to the rounding of P)."""
    exact = not (dtype == BF16 and d == 64)
    B, S, Hk, G = 2, 150, 2, 3
    q, k, v, dout = inputs(cuda_device, B, S, Hk, G, d, dtype, False, 21)
    slopes = torch.rand(Hk * G, device=cuda_device) if bias else None
    mask = mask_of(cuda_device, [list(range(S))] * B, None)
    got = run(q, k, v, dout, G, d ** -0.5, mask, softcap, slopes, False)
    assert int(torch.count_nonzero(got["dq"])) == 0 and (not exact or int(torch.count_nonzero(got["dk"])) == 0)
    want = ref.attention(q, k, v, dout, [list(range(S))] * B, None, G, d ** -0.5, softcap, slopes, False, dtype, dtype == BF16 and d == 64)
    for name in ("o", "lse", "dv", "dk"):
        ref.check(got[name], want[name], name)
    mixed = [[0] * 40 + list(range(1, 31)) + [31] * 80] * B
    mask = mask_of(cuda_device, mixed, None)
    got = run(q, k, v, dout, G, d ** -0.5, mask, softcap, slopes, False)
    assert int(torch.count_nonzero(got["dq"].view(B, Hk, G, S, d)[..., [0, 40, 55, 69, 70], :])) == 0
    assert not exact or int(torch.count_nonzero(got["dk"].view(B, Hk, S, d)[..., 40:70, :])) == 0
    want = ref.attention(q, k, v, dout, mixed, None, G, d ** -0.5, softcap, slopes, False, dtype, dtype == BF16)
    for name, value in want.items():
        ref.check(got[name], value, name)


def test_ids_of_64_bits(cuda_device):
    """Neighbouring documents whose ids agree in their low 32 bits are two, and so is a negative id whose low half is not."""
    ids = [0] * 5 + [1 << 32] * 7 + [(1 << 32) + 1] * 3 + [1] * 9 + [-(1 << 32) + 1] * 4 + [1] * 6 + [(1 << 63) - 1] * 8
    small = [0] * 5 + [1] * 7 + [2] * 3 + [3] * 9 + [-1] * 4 + [3] * 6 + [4] * 8
    n = 4 * len(ids)
    a, b = (mask_of(cuda_device, [x], None, torch.int64).block.view(torch.int32)[:n] for x in (ids, small))
    assert torch.equal(a, b)


def test_heads_beyond_2_to_the_31_elements(cuda_device):
    """33 heads of a million positions in documents of 100: offsets pass 32 bits in q, o and the gradients."""
    S, G, d, doc = 1 << 20, 33, 64, 100
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    ids = (torch.arange(S, device=cuda_device, dtype=torch.int32) // doc).view(1, S)
    rand = lambda *s: torch.randn(*s, device=cuda_device, generator=gen, dtype=BF16)  # noqa: E731
    q, k, v, dout = rand(1, G * S, d), rand(1, S, d), rand(1, S, d), rand(1, G * S, d)
    got = run(q, k, v, dout, G, 0.125, backend.attention_mask(ids), 0.0, None, False)
    for first in (0, (S // 2) // doc * doc, S // doc * doc - doc):
        part = lambda t, n: t.view(n, S, -1)[:, first:first + doc].reshape(1, n * doc, -1).contiguous()  # noqa: E731
        want = ref.attention(part(q, G), part(k, 1), part(v, 1), part(dout, G), [[0] * doc], None, G, 0.125, 0.0, None, False, BF16, True)
        for name, n in (("o", G), ("dq", G), ("dk", 1), ("dv", 1)):
            ref.check(part(got[name], n), want[name], f"{name} from {first}")
