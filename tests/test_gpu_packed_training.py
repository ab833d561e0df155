"""Layer norm, the embedding with its table's gradient and clipping by the global norm against float64, and a training step over packed
documents that runs them with masked attention.

Bounds: a float32 sum of n terms by threads and a tree of at most n / 32 + 40 additions a path is off by at most that many times 2^-24 of
the terms' magnitudes; a value stored in bfloat16 by 2^-8 of itself."""
import math

import numpy as np
import pytest
import torch

from metal_candle_b200 import backend, training
from metal_candle_b200.training import AdamW, AdamWConfig, GradClipper, clip_grad_norm, grad_norm
from tests.support import packed_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(dev, *shape, seed=0, dtype=F32, scale=1.0, shift=0.0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(*shape, device=dev, generator=gen) * scale + shift).to(dtype)


# ---- layer norm ------------------------------------------------------------------------------------------------------------

def layer_norm_64(x, w, b, dy, res, eps, dtype):
    """{name: (value, bound)}."""
    u = half_step(dtype)
    x, w, b, dy, res = (None if t is None else t.detach().cpu().double() for t in (x, w, b, dy, res))
    D = x.shape[-1]
    x, dy = x.reshape(-1, D), dy.reshape(-1, D)
    steps = (D / 32 + 40) * 2.0 ** -24
    mean = x.mean(-1, keepdim=True)
    off = x - mean
    var = (off * off).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    n = off * rstd
    dmean = steps * x.abs().mean(-1, keepdim=True)
    doff = dmean + 2.0 ** -24 * off.abs()
    dvar = 2 * (off.abs() * doff).mean(-1, keepdim=True) + steps * var
    dn = doff * rstd + n.abs() * (dvar / (2 * (var + eps)) + 2.0 ** -22)
    wv, bv = (torch.ones(D).double() if w is None else w), (torch.zeros(D).double() if b is None else b)
    y = n * wv + bv
    ey = dn * wv.abs() + 2.0 ** -22 * ((n * wv).abs() + bv.abs()) + u * y.abs()
    g = dy * wv
    a, q = g.mean(-1, keepdim=True), (g * n).mean(-1, keepdim=True)
    da = (steps + 2.0 ** -23) * g.abs().mean(-1, keepdim=True)
    dq = (steps + 2.0 ** -23) * (g * n).abs().mean(-1, keepdim=True) + (g.abs() * dn).mean(-1, keepdim=True)
    dx = (g - a - n * q) * rstd
    ex = rstd * (2.0 ** -23 * (g.abs() + a.abs() + (n * q).abs()) + da + dn * q.abs() + n.abs() * dq) + dx.abs() * (dvar / (2 * (var + eps)) + 2.0 ** -22)
    if res is not None:
        dx = dx + res.reshape(-1, D)
    ex = ex + u * dx.abs() + 2.0 ** -24 * dx.abs()
    rows = (x.shape[0] / 8 + 40) * 2.0 ** -24
    return dict(y=(y, ey), dx=(dx, ex), dw=((dy * n).sum(0), rows * (dy * n).abs().sum(0) + (dy.abs() * dn).sum(0)),
                db=(dy.sum(0), rows * dy.abs().sum(0)), mean=(mean[:, 0], dmean[:, 0] + 2.0 ** -23 * mean[:, 0].abs()),
                rstd=(rstd[:, 0], rstd[:, 0] * (dvar / (2 * (var + eps)) + 2.0 ** -22)[:, 0]))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (1, 7), (5, 64), (130, 128), (7, 777), (16, 896), (333, 896), (64, 1000), (9, 2048), (5, 2049), (4, 4096),
                                    (6, 8192), (3, 16384), (2, 20000), (3, 5001), (5000, 24), (2500, 40)])
def test_layer_norm(cuda_device, dtype, rows, D):
    x = rand(cuda_device, rows, D, seed=1, dtype=dtype, scale=2.0, shift=3.0)
    w, b, dy, res = (rand(cuda_device, *s, seed=i + 2, dtype=dtype) for i, s in enumerate([(D,), (D,), (rows, D), (rows, D)]))
    for full in (True, False):
        got = {}
        got["y"], got["mean"], got["rstd"] = backend.layer_norm_fused(x, w if full else None, b if full else None, 1e-5, return_stats=True)
        got["dx"], got["dw"], got["db"] = backend.layer_norm_backward(x, w if full else None, dy, 1e-5, dx_residual=res if full else None)
        want = layer_norm_64(x, w if full else None, b if full else None, dy, res if full else None, 1e-5, dtype)
        for name, value in want.items():
            ref.check(got[name], value, name)
    again = backend.layer_norm_backward(x, None, dy, 1e-5)
    assert all(torch.equal(a, got[n]) for a, n in zip(again, ("dx", "dw", "db")))
    only, none_w, none_b = backend.layer_norm_backward(x, None, dy, 1e-5, need_dw=False)
    assert torch.equal(only, got["dx"]) and none_w is None and none_b is None


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_of_a_large_mean(cuda_device, dtype):
    """The variance of rows whose mean is a thousand times their spread (E[x^2] - mean^2 would have no digit of it in float32)."""
    x = rand(cuda_device, 40, 512, seed=3, dtype=dtype, scale=8.0 if dtype == BF16 else 1.0, shift=2000.0)
    dy = rand(cuda_device, 40, 512, seed=4, dtype=dtype)
    want = layer_norm_64(x, None, None, dy, None, 1e-5, dtype)
    ref.check(backend.layer_norm_fused(x, eps=1e-5), want["y"], "y")
    ref.check(backend.layer_norm_backward(x, None, dy, 1e-5)[0], want["dx"], "dx")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_off_alignment_and_in_parts(cuda_device, dtype):
    """Buffers that start off a 16-byte boundary, and sums that go on over two calls."""
    rows, D = 70, 896
    flat = rand(cuda_device, 3 * rows * D + 8, seed=5, dtype=dtype)
    x, dy, res = (flat[1 + i * rows * D:1 + (i + 1) * rows * D].view(rows, D) for i in range(3))
    w = rand(cuda_device, D + 1, seed=6, dtype=dtype)[1:]
    want = layer_norm_64(x, w, None, dy, res, 1e-5, dtype)
    ref.check(backend.layer_norm_fused(x, w), want["y"], "y")
    dx, dw, db = backend.layer_norm_backward(x, w, dy, dx_residual=res)
    for name, t in (("dx", dx), ("dw", dw), ("db", db)):
        ref.check(t, want[name], name)
    half = rows // 2
    gw, gb = torch.zeros(D, device=cuda_device), torch.zeros(D, device=cuda_device)
    for part in (slice(0, half), slice(half, rows)):
        backend.layer_norm_backward(x[part].contiguous(), w, dy[part].contiguous(), grad_w=gw, grad_b=gb, accumulate=True)
    ref.check(gw, want["dw"], "dw in parts")
    ref.check(gb, want["db"], "db in parts")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("D,start", [(896, 0), (896, 3), (777, 0), (777, 5), (33, 1), (2500, 0)])
def test_layer_norm_in_place(cuda_device, dtype, D, start):
    """y over x, dx over dy and over the residual's gradient, for rows that start anywhere."""
    from metal_candle_b200 import _lib

    lib, rows, code = _lib.load(), 300, 0 if dtype == F32 else 1
    stream = torch.cuda.current_stream().cuda_stream
    flat = lambda seed: rand(cuda_device, rows * D + 8, seed=seed, dtype=dtype)[start:start + rows * D].view(rows, D)  # noqa: E731
    x, dy, res, w, b = flat(1), flat(2), flat(3), rand(cuda_device, D, seed=4, dtype=dtype), rand(cuda_device, D, seed=5, dtype=dtype)
    want = layer_norm_64(x, w, b, dy, res, 1e-5, dtype)
    ws = torch.empty(lib.mcb_layernorm_bwd_workspace_bytes(rows, D), dtype=torch.uint8, device=cuda_device)
    for over in ("dy", "res"):
        d, r, dw, db = dy.clone(), res.clone(), torch.empty(D, device=cuda_device), torch.empty(D, device=cuda_device)
        dc, rc = (torch.empty(rows * D + 8, dtype=dtype, device=cuda_device)[start:start + rows * D].view(rows, D) for _ in range(2))
        dc.copy_(d), rc.copy_(r)
        out = dc if over == "dy" else rc
        _lib.check(lib.mcb_layernorm_bwd(x.data_ptr(), w.data_ptr(), dc.data_ptr(), rc.data_ptr(), out.data_ptr(), dw.data_ptr(), db.data_ptr(), 0, rows, D,
                                         1e-5, code, ws.data_ptr(), ws.numel(), stream))
        for name, t in (("dx", out), ("dw", dw), ("db", db)):
            ref.check(t, want[name], f"{name} over {over}")
        # one of the two sums alone
        only = torch.empty(D, device=cuda_device)
        _lib.check(lib.mcb_layernorm_bwd(x.data_ptr(), w.data_ptr(), d.data_ptr(), None, torch.empty_like(d).data_ptr(), None, only.data_ptr(), 0, rows, D,
                                         1e-5, code, ws.data_ptr(), ws.numel(), stream))
        ref.check(only, want["db"], "db alone")
    _lib.check(lib.mcb_layernorm_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), x.data_ptr(), None, None, rows, D, 1e-5, code, stream))
    ref.check(x, want["y"], "y over x")


# ---- embedding -------------------------------------------------------------------------------------------------------------

def embedding_64(ids, dout, vocab, scale):
    ids, dout = ids.cpu().reshape(-1), dout.detach().cpu().double().reshape(ids.numel(), -1)
    keep = (ids >= 0) & (ids < vocab)
    at, rows = ids[keep].long(), dout[keep] * float(np.float32(scale))
    grad = torch.zeros(vocab, dout.shape[1], dtype=torch.float64).index_add_(0, at, rows)
    size = torch.zeros_like(grad).index_add_(0, at, rows.abs())
    count = torch.bincount(at, minlength=vocab).double()[:, None]
    return grad, (32 + count / 32 + 3) * 2.0 ** -24 * size


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,H,V,kind", [(1, 1, 1, "any"), (2, 3, 5, "any"), (17, 128, 1000, "any"), (33, 896, 151936, "any"), (64, 7, 2, "any"), (1024, 40, 511, "any"),
                                        (1025, 24, 512, "any"), (3000, 64, 300000, "any"), (5000, 100, 50, "any"), (9000, 16, 4097, "one"), (700, 32, 100, "none"),
                                        (20000, 8, 30000, "hot"), (4097, 1030, 9, "any")])
def test_embedding(cuda_device, dtype, M, H, V, kind):
    gen = torch.Generator(device=cuda_device).manual_seed(M)
    ids = torch.randint(-1, V + 1, (M,), device=cuda_device, generator=gen)   # one below and one above as well
    if kind == "one":
        ids.fill_(V - 1)
    elif kind == "none":
        ids.fill_(-1)
    elif kind == "hot":
        ids = torch.where(torch.rand(M, device=cuda_device, generator=gen) < 0.5, torch.full_like(ids, 7), ids)
    table, dout = rand(cuda_device, V, H, seed=1, dtype=dtype), rand(cuda_device, M, H, seed=2, dtype=dtype)
    scale = 29.933
    keep = (ids >= 0) & (ids < V)
    for index in (ids, ids.to(torch.int32)):
        out = backend.embedding(index, table, scale)
        want = torch.where(keep[:, None], (table.float() * np.float32(scale))[ids.clamp(0, V - 1)], torch.zeros((), device=cuda_device)).to(dtype)
        assert torch.equal(out, want)
        grad = backend.embedding_backward(index, dout, V, scale)
        value = embedding_64(ids, dout, V, scale)
        ref.check(grad, value, "grad")
        assert torch.equal(grad, backend.embedding_backward(index, dout, V, scale))
    # added to what is there; rows that no token names are left alone
    before = rand(cuda_device, V, H, seed=3)
    more = backend.embedding_backward(ids, dout, V, scale, grad=before.clone(), accumulate=True)
    ref.check(more, (before.cpu().double() + value[0], value[1] + 2.0 ** -24 * (before.cpu().double().abs() + value[0].abs())), "accumulated")
    named = torch.zeros(V, dtype=torch.bool, device=cuda_device)
    named[ids[keep]] = True
    assert torch.equal(more[~named], before[~named])
    assert (grad[~named] == 0).all()


def test_embedding_of_any_shape_and_alignment(cuda_device):
    ids = torch.tensor([[3, 1, -1], [1, 9, 3]], device=cuda_device)
    flat = rand(cuda_device, 2 * 3 * 16 + 1, seed=1, dtype=BF16)
    dout = flat[1:].view(2, 3, 16)
    table = rand(cuda_device, 10 * 16 + 3, seed=2, dtype=BF16)[3:].view(10, 16)
    out = backend.embedding(ids, table)
    assert out.shape == (2, 3, 16) and torch.equal(out[0, 1], table[1]) and (out[0, 2] == 0).all()
    ref.check(backend.embedding_backward(ids, dout, 10), embedding_64(ids, dout, 10, 1.0), "grad")
    # values that are not finite stay in their own rows
    dout = dout.clone()
    dout[0, 0] = math.nan
    grad = backend.embedding_backward(ids, dout, 10)
    assert torch.isnan(grad[3]).all() and torch.isfinite(grad[[0, 1, 2, 4, 5, 6, 7, 8, 9]]).all()


# ---- global norm -----------------------------------------------------------------------------------------------------------

def norm_64(tensors):
    return math.sqrt(sum(float(t.double().square().sum()) for t in tensors))


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [4096, 4097, 1], [17] * 600, [100003, 1, 8192], [1 << 22]])
@pytest.mark.parametrize("dtype", [F32, BF16, None])
def test_norm_and_clip(cuda_device, sizes, dtype):
    grads = [rand(cuda_device, n, seed=i, dtype=dtype or (BF16 if i % 2 else F32)) for i, n in enumerate(sizes)]
    whole = norm_64(grads)
    # at most 16 float32 additions of squares a thread, the rest in float64, and the root's rounding
    near = lambda got, want: abs(float(got) - want) <= 17 * 2.0 ** -24 * want  # noqa: E731
    assert near(grad_norm(grads), whole)
    for limit in (whole / 3, whole * 3, 0.0, math.inf):
        out = [torch.full_like(g, 7.0) for g in grads]
        copies = [g.clone() for g in grads]
        clipper = GradClipper(copies, out=out)
        assert near(clipper.clip(limit), whole)
        factor = np.float32(1.0)
        if limit != math.inf:
            factor = min(np.float32(1.0), np.float32(limit) / (np.float32(float(grad_norm(grads))) + np.float32(1e-6)))
        for g, o, c in zip(grads, out, copies):
            assert torch.equal(g, c)
            want = g.double() * float(factor)
            # the factor's own rounding (division and sum: three half steps) and the product's
            assert ((o.double() - want).abs() <= (2.0 ** -22 + half_step(g.dtype)) * want.abs() + 1e-44).all()
        assert near(clip_grad_norm(copies, limit), whole)
        assert all(torch.equal(o, c) for o, c in zip(out, copies))


def test_norm_of_nothing(cuda_device):
    empty = [torch.empty(0, device=cuda_device), torch.empty(0, 5, dtype=BF16, device=cuda_device)]
    assert float(grad_norm(empty)) == 0.0 and float(clip_grad_norm(empty, 1.0)) == 0.0


def test_norm_at_the_ends_of_float32(cuda_device):
    for value in (3e38, 1e25, 1e-30, 1e-42):
        g = torch.full((5000,), value, device=cuda_device)
        g[1] = 0.0
        want = norm_64([g])
        if want < 3.4e38:
            assert abs(float(grad_norm([g])) - want) <= 2.0 ** -22 * want + 1e-45
        else:
            assert float(grad_norm([g])) == math.inf
    g = rand(cuda_device, 5000, seed=1)
    for bad in (math.nan, math.inf):
        x = g.clone()
        x[4999] = bad
        norm = float(grad_norm([g, x]))
        assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
        clipped = [g.clone(), x]
        clip_grad_norm(clipped, 1.0)
        # NaN everywhere, or 0 for what was finite (and NaN for inf * 0)
        assert torch.isnan(clipped[0]).all() if math.isnan(bad) else (clipped[0] == 0).all() and torch.isnan(x[4999])


def test_clip_off_alignment(cuda_device):
    for dtype in (F32, BF16):
        flat = rand(cuda_device, 20011, seed=1, dtype=dtype)
        grads = [flat[1:4000], flat[4001:4002], flat[4005:20011]]
        want = norm_64(grads)
        out = torch.zeros(20011, dtype=dtype, device=cuda_device)
        norm = clip_grad_norm(grads, 1.0, out=[out[1:4000], out[4001:4002], out[4005:20011]])
        assert abs(float(norm) - want) <= 2.0 ** -19 * want
        mine = flat.double() / want
        mine[0], mine[4000], mine[4002:4005] = 0, 0, 0
        assert ((out.double() - mine).abs() <= (2.0 ** -18 + half_step(dtype)) * mine.abs() + 1e-8).all()


@pytest.mark.parametrize("count", [3, 200, 700])
def test_adamw_clipped_is_clip_then_adamw(cuda_device, count):
    """The same bits as clipping the gradients first, with the gradients left alone; the limit at work and not."""
    config = AdamWConfig(learning_rate=1e-2)
    for limit in (0.5, 1e9):
        params = [rand(cuda_device, 5 + 13 * (i % 50), seed=i) for i in range(count)]
        grads = [rand(cuda_device, 5 + 13 * (i % 50), seed=1000 + i) for i in range(count)]
        one, two = [p.clone() for p in params], [p.clone() for p in params]
        a, b = AdamW(config), AdamW(config)
        for _ in range(2):
            norm = a.step_vars(one, grads, max_grad_norm=limit)
            clipped = [g.clone() for g in grads]
            assert torch.equal(norm, clip_grad_norm(clipped, limit))
            assert b.step_vars(two, clipped) is None
            assert all(torch.equal(x, y) for x, y in zip(one, two))
        # a scale in front of the gradients counts in the norm
        scaled = a.step_vars(one, grads, grad_scale=0.25, max_grad_norm=limit)
        assert abs(float(scaled) - 0.25 * float(norm)) <= 2.0 ** -22 * float(norm)


def test_trainer_clips_where_it_is_told_to(cuda_device):
    """TrainingConfig.clip_gradients makes max_grad_norm count; without it nothing changes."""
    def train(**config):
        gen = torch.Generator(device=cuda_device).manual_seed(3)
        t = training.Trainer(32, 64, 1, training.LoRAAdapterConfig(rank=4), training.TrainingConfig(num_epochs=1, **config), cuda_device, generator=gen)
        n = len(training.TrainingStep.collect_trainable_vars(t.lora_adapter()))

        def step(ids, targets):
            return 1.0, [torch.full_like(v, 10.0) for v in training.TrainingStep.collect_trainable_vars(t.lora_adapter())]

        t.train([(None, None)] * 2, step, verbose=False)
        assert n == 4
        return [(m, v) for m, v in t.optimizer.state.values()]

    plain, off, on = train(), train(max_grad_norm=1e-3), train(max_grad_norm=1e-3, clip_gradients=True)
    assert all(torch.equal(a, b) for p, o in zip(plain, off) for a, b in zip(p, o))
    assert all(float(o[0].abs().max()) < 1e-3 < float(p[0].abs().max()) for p, o in zip(plain, on))


# ---- streams, graphs -------------------------------------------------------------------------------------------------------

def test_captured_and_on_other_streams(cuda_device):
    x, w, b, dy = (rand(cuda_device, *s, seed=i) for i, s in enumerate([(300, 96), (96,), (96,), (300, 96)]))
    ids = torch.randint(0, 50, (300,), device=cuda_device)
    grads = [rand(cuda_device, 3000, seed=7), rand(cuda_device, 11, seed=8)]
    clipped = [torch.empty_like(g) for g in grads]
    clipper = GradClipper(grads, out=clipped)

    def step():
        return [backend.layer_norm_fused(x, w, b), *backend.layer_norm_backward(x, w, dy), backend.embedding(ids, dy[:50], 2.0),
                backend.embedding_backward(ids, dy, 50, 2.0), clipper.clip(1.0), *[c.clone() for c in clipped]]

    want = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for t in (x, dy, grads[0]):
        t.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(held, step()))
    assert not torch.equal(held[0], want[0])


# ---- a run of them together --------------------------------------------------------------------------------------------------

def test_a_training_step_over_packed_documents(cuda_device):
    """Embedding, layer norm, masked attention, a squared loss, their gradients, and AdamW with clipping: the step that autograd in
    float64 takes."""
    B, S, H, V, heads, d = 2, 45, 48, 60, 3, 16
    dev = cuda_device
    ids = torch.randint(0, V, (B, S), generator=torch.Generator().manual_seed(1))
    docs = torch.tensor([[0] * 20 + [1] * 22 + [-1] * 3, [2] * 45], dtype=torch.int32)
    ids[docs < 0] = -1
    table, w, b, target = rand(dev, V, H, seed=1), 1 + 0.1 * rand(dev, H, seed=2), 0.1 * rand(dev, H, seed=3), rand(dev, B * S, H, seed=4)
    slopes, scale, emb_scale, limit = torch.tensor([0.5, 0.1, 0.02], device=dev), 0.25, 6.9, 0.5
    # the framework's
    mask = backend.attention_mask(docs.to(dev))
    x = backend.embedding(ids.to(dev), table, emb_scale).view(B * S, H)
    n = backend.layer_norm_fused(x, w, b)
    split = n.view(B, S, heads, d).permute(0, 2, 1, 3).reshape(B * heads, S, d).contiguous()
    how = dict(groups=1, scale=scale, mask=mask, softcap=8.0, slopes=slopes, token_major=True)
    o, lse = backend.attention_masked_forward(split, split, split, **how)
    keep = (docs >= 0).reshape(-1, 1).to(dev)
    dout = torch.where(keep, o - target, torch.zeros((), device=dev))
    dn = sum(backend.attention_masked_backward(split, split, split, o, lse, dout, **how)).view(B, heads, S, d).permute(0, 2, 1, 3).reshape(B * S, H)
    dx, dw, db = backend.layer_norm_backward(x, w, dn.contiguous())
    dtable = backend.embedding_backward(ids.to(dev), dx.view(B, S, H), V, emb_scale)
    params, grads = [table.clone(), w.clone(), b.clone()], [dtable, dw, db]
    optimizer = AdamW(AdamWConfig(learning_rate=1e-2))
    norm = optimizer.step_vars(params, grads, max_grad_norm=limit)
    # autograd's
    t64, w64, b64 = (t.detach().cpu().double().requires_grad_(True) for t in (table, w, b))
    rows = torch.where((ids >= 0)[..., None], t64[ids.clamp_min(0)] * float(np.float32(emb_scale)), torch.zeros((), dtype=torch.float64)).view(B * S, H)
    var, mean = torch.var_mean(rows, -1, correction=0, keepdim=True)
    y = ((rows - mean) / torch.sqrt(var + 1e-5) * w64 + b64).view(B, S, heads, d).permute(0, 2, 1, 3)
    at = torch.arange(S).double()
    s = 8.0 * torch.tanh(y @ y.transpose(-1, -2) * scale / 8.0) - slopes.cpu().double().view(1, heads, 1, 1) * (at[:, None] - at[None, :]).abs()
    see = torch.stack([ref.visible(r.tolist(), None) for r in docs])[:, None]
    p = torch.softmax(s.masked_fill(~see, -1e300), -1) * see
    out = (p @ y).permute(0, 2, 1, 3).reshape(B * S, H)
    loss = (0.5 * (out - target.cpu().double()).square() * (docs >= 0).reshape(-1, 1)).sum()
    want = torch.autograd.grad(loss, (t64, w64, b64))
    # some 500 float32 roundings on the way to a gradient, none of which a value of order 1 amplifies by more than 10 or so
    for got, exact in zip(grads, want):
        assert (got.cpu().double() - exact).norm() <= 500 * 10 * 2.0 ** -24 * exact.norm()
    whole = norm_64(want)
    assert abs(float(norm) - whole) <= 500 * 10 * 2.0 ** -24 * whole
    # AdamW from zero moments; the counter is shared, so tensor j of the step has the bias corrections of step j + 1.  Where a gradient is
    # not tiny its size cancels, and what is left are float32 roundings of order 1e-2
    factor = min(1.0, limit / (whole + 1e-6))
    for j, (before, after, exact) in enumerate(zip((table, w, b), params, want)):
        g = exact * factor
        moment, square = 0.1 * g / (1 - 0.9 ** (j + 1)), 0.001 * g * g / (1 - 0.999 ** (j + 1))
        step = 1e-2 * moment / (square.sqrt() + 1e-8) + 1e-2 * 0.01 * before.cpu().double()
        clear = g.abs() > 1e-4
        assert clear.any() and ((before - after).cpu().double() - step)[clear].abs().max() <= 1e-5


def test_chained_launches_change_nothing(cuda_device):
    """Kernels launched while the one before still runs, against launches that wait for it: every call reads what the last one wrote."""
    from metal_candle_b200 import _lib

    lib = _lib.load()
    B, S, Hk, G, d, V = 2, 300, 2, 3, 64, 500
    D = Hk * G * d
    gen = torch.Generator(device=cuda_device).manual_seed(8)
    ids = torch.randint(-1, V, (B, S), device=cuda_device, generator=gen, dtype=torch.int32)
    docs = (torch.arange(S, device=cuda_device) // 70).expand(B, S).contiguous()
    begin = {dtype: (rand(cuda_device, V, D, seed=1, dtype=dtype), rand(cuda_device, D, seed=2, dtype=dtype)) for dtype in (BF16, F32)}

    def chain():
        out = []
        for dtype, (table, w) in begin.items():
            for _ in range(2):
                mask = backend.attention_mask(docs)
                x = backend.embedding(ids, table, 2.0).view(B * S, D)
                n = backend.layer_norm_fused(x, w, w)
                q = n.view(B * Hk, G * S, d)
                k = q[:, :S].contiguous()
                how = dict(groups=G, scale=0.125, mask=mask, token_major=True)
                o, lse = backend.attention_masked_forward(q, k, k, **how)
                dq, dk, dv = backend.attention_masked_backward(q, k, k, o, lse, n, **how)
                dx, dw, db = backend.layer_norm_backward(x, w, dq.view(B * S, D), dx_residual=n)
                grad = backend.embedding_backward(ids, dx.view(B, S, D), V, 2.0)
                norm = clip_grad_norm([grad, dw, db, dk, dv], 1.0)
                table, w = grad.to(dtype), (w + dw.to(dtype))
                out += [o, lse, dq, dk, dv, dx, dw, db, grad, norm]
        return out

    try:
        _lib.check(lib.mcb_set_option(_lib.MCB_OPT_PDL, 0))
        want = chain()
        torch.cuda.synchronize()
    finally:
        _lib.check(lib.mcb_set_option(_lib.MCB_OPT_PDL, 1))
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(chain(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = chain()
    for _ in range(3):
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_ids_of_64_bits_and_rows_beyond_2_to_the_31_elements(cuda_device):
    """Ids whose low 32 bits alone would be in the vocabulary are outside it; a table of more than 2^31 elements is reached to its end."""
    V, H = 600_001, 3600
    table = torch.zeros(V, H, dtype=BF16, device=cuda_device)
    table[V - 1] = rand(cuda_device, H, seed=1, dtype=BF16)
    table[7] = 3.0
    ids = torch.tensor([V - 1, 7, (1 << 32) + 7, -(1 << 32) + 7, V, V - 1, -1], device=cuda_device)
    out = backend.embedding(ids, table, 2.0)
    assert torch.equal(out[0], table[V - 1] * 2) and torch.equal(out[5], out[0]) and (out[1] == 6.0).all()
    assert (out[[2, 3, 4, 6]] == 0).all()
    del table
    grad = torch.full((V, H), math.nan, device=cuda_device)
    dout = rand(cuda_device, 7, H, seed=2)
    backend.embedding_backward(ids, dout, V, 1.0, grad=grad)
    assert torch.equal(grad[V - 1], dout[0] + dout[5]) and torch.equal(grad[7], dout[1])
    grad[V - 1], grad[7] = 0.0, 0.0
    assert all(int(torch.count_nonzero(part)) == 0 for part in grad.split(100_000))


def test_layer_norm_beyond_2_to_the_31_elements(cuda_device):
    rows, D = 2_400_000, 904
    x = torch.empty(rows, D, dtype=BF16, device=cuda_device)
    head, tail = rand(cuda_device, 300, D, seed=1, dtype=BF16), rand(cuda_device, 300, D, seed=2, dtype=BF16)
    x.zero_()
    x[:300], x[-300:] = head, tail
    dy = torch.zeros_like(x)
    dy[:300], dy[-300:] = tail, head
    w = rand(cuda_device, D, seed=3, dtype=BF16)
    y = backend.layer_norm_fused(x, w, w)
    dx, dw, db = backend.layer_norm_backward(x, w, dy)
    want = layer_norm_64(torch.cat([head, tail]), w, w, torch.cat([tail, head]), None, 1e-5, BF16)
    ref.check(torch.cat([y[:300], y[-300:]]), want["y"], "y")
    ref.check(torch.cat([dx[:300], dx[-300:]]), want["dx"], "dx")
    for name, t in (("dw", dw), ("db", db)):   # rows of zeros add exact zeros: the sums are those of the 600 rows, in another order
        ref.check(t, want[name], name)


def test_clipping_beyond_2_to_the_31_elements(cuda_device):
    n = (1 << 31) + 4099
    g = torch.zeros(n, dtype=BF16, device=cuda_device)
    g[0], g[1 << 31], g[-1] = 2.0, 6.0, 9.0
    assert abs(float(clip_grad_norm([g], 1.1)) - 11.0) <= 11 * 2.0 ** -23
    f = torch.tensor([2.0, 6.0, 9.0], dtype=BF16) * (1.1 / (11 + 1e-6))   # (a tenth of each, to a rounding of bfloat16)
    got = torch.stack([g[0], g[1 << 31], g[-1]]).cpu()
    assert ((got.float() - f.float()).abs() <= 2 * 2.0 ** -8 * f.float()).all()
    assert int(torch.count_nonzero(g)) == 3
