"""What the entry points of training on packed documents refuse, on the CPU: nothing is launched, no pointer is followed."""
import ctypes as C
import math

import pytest
import torch

from metal_candle_b200 import _lib, backend, training
from metal_candle_b200.backend import TrainingError
from metal_candle_b200.training import InvalidConfig

NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, NOT_INIT = -1, -2, -3, -4, -5, -6
F32, BF16 = _lib.MCB_F32, _lib.MCB_BF16
HUGE = 1 << 40


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_mask(lib):
    assert lib.mcb_attention_mask_bytes(2, 4096) % 16 == 0 and lib.mcb_attention_mask_bytes(2, 4096) > 4 * 8 * 4096
    for batch, seq in ((0, 1), (1, 0), (65536, 1), (1, 1 << 30), (4, 1 << 29)):
        assert lib.mcb_attention_mask_bytes(batch, seq) == 0
    ok = dict(ids=16, id_bytes=4, prefix=None, mask=16, nbytes=HUGE, batch=2, seq=10)

    def call(**change):
        a = {**ok, **change}
        return lib.mcb_attention_mask(a["ids"], a["id_bytes"], a["prefix"], a["mask"], a["nbytes"], a["batch"], a["seq"], None)

    assert call(mask=None) == NULL and call(batch=0) == SHAPE and call(seq=1 << 30) == SHAPE and call(id_bytes=2) == UNSUPPORTED
    assert call(mask=24) == ALIGN and call(ids=18) == ALIGN and call(ids=20, id_bytes=8) == ALIGN
    assert call(nbytes=lib.mcb_attention_mask_bytes(2, 10) - 1) == WORKSPACE


def attention(**change):
    a = dict(mask=16, mask_bytes=HUGE, slopes=None, batch=2, seq=100, kv_heads=2, groups=3, head_dim=64, scale=0.125, softcap=0.0, dtype=BF16,
             o_token_major=0)
    a.update(change)
    return _lib.MaskedAttention(**a)


REFUSED = [(dict(mask=None), NULL), (dict(dtype=2), UNSUPPORTED), (dict(seq=0), SHAPE), (dict(batch=0), SHAPE), (dict(mask_bytes=64), SHAPE),
           (dict(head_dim=0), UNSUPPORTED), (dict(head_dim=4), UNSUPPORTED), (dict(head_dim=60), UNSUPPORTED), (dict(head_dim=136), UNSUPPORTED),
           (dict(kv_heads=0), SHAPE), (dict(groups=0), SHAPE), (dict(kv_heads=1 << 20, groups=1 << 20), SHAPE), (dict(groups=1 << 26), SHAPE),
           (dict(scale=math.nan), SHAPE), (dict(scale=math.inf), SHAPE), (dict(scale=0.0), SHAPE),
           (dict(scale=-0.1), SHAPE), (dict(softcap=-1.0), SHAPE), (dict(softcap=math.nan), SHAPE),
           (dict(softcap=math.inf), SHAPE), (dict(softcap=3e38), SHAPE), (dict(softcap=1e-42), SHAPE), (dict(scale=3e38), SHAPE), (dict(mask=24), ALIGN), (dict(slopes=17), ALIGN)]


@pytest.mark.parametrize("change,status", REFUSED)
def test_attention(lib, change, status):
    call = attention(**change)
    assert lib.mcb_attention_masked_fwd(C.byref(call), 16, 16, 16, 16, None, None) == status
    assert lib.mcb_attention_masked_bwd(C.byref(call), 16, 16, 16, 16, 16, 16, 16, 16, 16, 1024, HUGE, None) == status
    assert lib.mcb_attention_masked_workspace_bytes(C.byref(call)) == 0


def test_attention_pointers(lib):
    call = attention()
    assert lib.mcb_attention_masked_fwd(None, 16, 16, 16, 16, None, None) == NULL
    for i in range(4):
        for value, status in ((None, NULL), (24, ALIGN)):
            args = [(i + 2) << 41 for i in range(4)]
            args[i] = value
            assert lib.mcb_attention_masked_fwd(C.byref(call), *args, None, None) == status
    for i in range(9):
        args = [(i + 2) << 41 for i in range(9)]
        args[i] = None
        assert lib.mcb_attention_masked_bwd(C.byref(call), *args, 1 << 50, HUGE, None) == NULL
        args[i] = 24 + (1 << 52)
        assert lib.mcb_attention_masked_bwd(C.byref(call), *args, 1 << 50, HUGE, None) == (ALIGN if i != 4 else NOT_INIT)   # lse is float32
    need = lib.mcb_attention_masked_workspace_bytes(C.byref(call))
    assert need >= 2 * 2 * 2 * 3 * 100 * 4
    for ws, n in ((None, HUGE), (1024, need - 1), (1040, HUGE)):
        assert lib.mcb_attention_masked_bwd(C.byref(call), *[(i + 2) << 41 for i in range(9)], ws, n, None) == WORKSPACE


def test_attention_outputs_overlap_nothing(lib):
    call = attention()
    size = 2 * 2 * 3 * 100 * 64 * (4 if call.dtype == 0 else 2)   # of q
    assert size == call.batch * call.kv_heads * call.groups * call.seq * call.head_dim * (4 if call.dtype == 0 else 2)
    far = [(i + 2) << 41 for i in range(9)]
    fwd = lambda *a: lib.mcb_attention_masked_fwd(C.byref(call), *a, None)                 # noqa: E731
    bwd = lambda *a: lib.mcb_attention_masked_bwd(C.byref(call), *a, 1 << 50, HUGE, None)   # noqa: E731
    assert fwd(*far[:5]) == bwd(*far) == NOT_INIT
    for other in (far[0], far[1], far[2]):
        assert fwd(*far[:3], other, far[4]) == SHAPE and fwd(*far[:4], other + 16) == SHAPE
    assert fwd(far[0], far[1], far[2], far[0] + size - 16, None) == SHAPE and fwd(far[0], far[1], far[2], far[0] + size, None) == NOT_INIT
    assert fwd(far[0], far[1], far[2], far[0] - size, None) == NOT_INIT
    for out in (6, 7, 8):
        for i in range(9):
            args = list(far)
            args[out] = args[i]
            assert bwd(*args) == (NOT_INIT if i == out else SHAPE)
    assert lib.mcb_attention_masked_bwd(C.byref(call), *far, far[0], HUGE, None) == SHAPE


def test_layer_norm(lib):
    def fwd(x=16, y=16, rows=4, D=8, eps=1e-5, dtype=F32):
        return lib.mcb_layernorm_fwd(x, None, None, y, None, None, rows, D, eps, dtype, None)

    def bwd(x=16, dy=16, dx=16, dw=16, db=16, rows=4, D=8, eps=1e-5, dtype=F32, ws=16, n=HUGE):
        return lib.mcb_layernorm_bwd(x, None, dy, None, dx, dw, db, 0, rows, D, eps, dtype, ws, n, None)

    for call in (fwd, bwd):
        assert call(x=None) == NULL and call(rows=0) == SHAPE and call(D=0) == SHAPE and call(D=1 << 30) == SHAPE and call(dtype=7) == UNSUPPORTED
        assert call(eps=-1.0) == SHAPE and call(eps=math.nan) == SHAPE and call(eps=math.inf) == SHAPE
    assert fwd(y=None) == NULL and bwd(dy=None) == NULL and bwd(dx=None) == NULL
    need = lib.mcb_layernorm_bwd_workspace_bytes(4, 8)
    assert need == 8 * 2 * 8 * 4 and lib.mcb_layernorm_bwd_workspace_bytes(0, 8) == 0
    assert bwd(ws=None) == WORKSPACE and bwd(n=need - 1) == WORKSPACE and bwd(ws=20) == WORKSPACE and bwd(dw=None, ws=None) == WORKSPACE


def test_embedding(lib):
    def fwd(ids=16, id_bytes=4, table=16, out=16, M=4, H=8, vocab=10, scale=1.0, dtype=F32):
        return lib.mcb_embedding_scaled_fwd(ids, id_bytes, table, out, M, H, vocab, scale, dtype, None)

    def bwd(ids=16, id_bytes=4, table=16, out=16, M=4, H=8, vocab=10, scale=1.0, dtype=F32, ws=16, n=HUGE):
        return lib.mcb_embedding_bwd(ids, id_bytes, table, out, 0, M, H, vocab, scale, dtype, ws, n, None)

    for call in (fwd, bwd):
        assert call(ids=None) == NULL and call(table=None) == NULL and call(out=None) == NULL
        assert call(id_bytes=1) == UNSUPPORTED and call(dtype=5) == UNSUPPORTED and call(scale=math.inf) == SHAPE and call(scale=math.nan) == SHAPE
        for change in (dict(M=0), dict(H=0), dict(vocab=0), dict(M=1 << 30), dict(H=1 << 23), dict(vocab=1 << 30)):
            assert call(**change) == SHAPE
    assert bwd(out=24) == ALIGN
    need = lib.mcb_embedding_bwd_workspace_bytes(4, 8)
    assert need == 4 * 256 + 2 * 8 * 4 and lib.mcb_embedding_bwd_workspace_bytes(0, 8) == 0
    assert bwd(ws=None) == WORKSPACE and bwd(n=need - 1) == WORKSPACE and bwd(ws=24) == WORKSPACE


def grads(*entries):
    """(g, out, n[, dtype]) each."""
    return (_lib.GradTensor * len(entries))(*[_lib.GradTensor(e[0], e[1], e[2], e[3] if len(e) > 3 else F32, 0) for e in entries])


def test_norm_and_clip(lib):
    good = grads((16, None, 10), (64, None, 3))
    norm = lambda t, n, out=16, ws=16, size=HUGE: lib.mcb_grad_norm(t, n, out, ws, size, None)  # noqa: E731
    clip = lambda t, n, limit=1.0, ws=16, size=HUGE: lib.mcb_clip_grad_norm(t, n, limit, None, ws, size, None)  # noqa: E731
    for call in (norm, clip):
        assert call(good, 0) == SHAPE and call(good, -1) == SHAPE and call(None, 2) == NULL
        assert call(grads((None, None, 1)), 1) == NULL and call(grads((16, None, -1)), 1) == SHAPE and call(grads((16, None, 1, 3)), 1) == UNSUPPORTED
        assert call(grads((18, None, 1)), 1) == ALIGN and call(grads((17, None, 1, BF16)), 1) == ALIGN
        assert call(good, 2, ws=None) == WORKSPACE and call(good, 2, ws=20) == WORKSPACE
        assert call(good, 2, size=lib.mcb_grad_norm_workspace_bytes(2) - 1) == WORKSPACE
    assert norm(good, 2, out=None) == NULL
    for limit in (-1.0, math.nan):
        assert clip(good, 2, limit) == SHAPE
    assert lib.mcb_grad_norm_workspace_bytes(513) == 2 * lib.mcb_grad_norm_workspace_bytes(512)
    assert clip(good, 2) == NOT_INIT and norm(grads((16, None, 4), (16, None, 4)), 2) == NOT_INIT   # (reading one twice is no harm)
    # what one block would write and another read: a tensor twice, overlapping ones, an output over another gradient or half its own
    for bad in (grads((16, None, 4), (16, None, 4)), grads((16, None, 8), (40, None, 8)), grads((16, 1024, 4), (1024, 2048, 4)),
                grads((16, 32, 8)), grads((16, 1024, 4), (64, 1028, 4)), grads((1024, None, 100), (4096, 1100, 2), (8192, None, 1))):
        assert clip(bad, len(bad)) == SHAPE
    assert clip(grads((16, 16, 4), (32, None, 4), (48, 1024, 4)), 3) == NOT_INIT


def test_adamw_clipped(lib):
    table = (_lib.AdamWTensor * 1)(_lib.AdamWTensor(16, 16, 16, 16, 4, 1, 0))

    def call(limit=1.0, ws=16, size=HUGE, beta1=0.9):
        return lib.mcb_adamw_multi_clipped(table, 1, 1e-3, beta1, 0.999, 1e-8, 0.0, 1.0, limit, None, ws, size, None)

    assert call(limit=-1.0) == SHAPE and call(limit=math.nan) == SHAPE and call(ws=None) == WORKSPACE and call(ws=24) == WORKSPACE
    assert call(size=lib.mcb_grad_norm_workspace_bytes(1) - 1) == WORKSPACE
    assert call(beta1=1.0) == SHAPE and lib.mcb_adamw_multi_clipped(None, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 1.0, None, 16, HUGE, None) == NULL


def test_host_layer():
    """Messages before anything reaches a device."""
    x = torch.zeros(4, 8)
    for call in (lambda: backend.layer_norm_fused(x), lambda: backend.layer_norm_backward(x, None, x), lambda: backend.embedding(torch.zeros(2, dtype=torch.int64), x),
                 lambda: backend.embedding_backward(torch.zeros(4, dtype=torch.int64), x, 10), lambda: backend.attention_mask(torch.zeros(1, 4, dtype=torch.int32)),
                 lambda: backend.attention_mask(batch=1, seq=4, device="cpu"), lambda: training.grad_norm([x]), lambda: training.clip_grad_norm([x], 1.0)):
        with pytest.raises(TrainingError, match="CUDA device"):
            call()
    meta = torch.zeros(4, 8, device="meta")
    for call, message in (
            (lambda: backend.layer_norm_fused(torch.zeros(4, 0)), "empty"), (lambda: backend.layer_norm_fused(x.half()), "unsupported dtype"),
            (lambda: backend.embedding(torch.zeros(2), x), "ids are"), (lambda: backend.embedding(torch.zeros(0, dtype=torch.int64), x), "empty ids"),
            (lambda: backend.embedding(torch.zeros(2, dtype=torch.int64), x[0]), "table must be"),
            (lambda: backend.embedding_backward(torch.zeros(3, dtype=torch.int64), x, 10), "does not fit"),
            (lambda: backend.embedding_backward(torch.zeros(4, dtype=torch.int64), x, 10, accumulate=True), "accumulate needs"),
            (lambda: backend.embedding_backward(torch.zeros(4, dtype=torch.int64), x, 10, grad=torch.zeros(9, 8)), "grad must be"),
            (lambda: backend.attention_mask(), "needs document_ids"), (lambda: backend.attention_mask(torch.zeros(4, dtype=torch.int32)), "are \\[batch, seq\\]"),
            (lambda: backend.attention_mask(torch.zeros(1, 4)), "document_ids is"),
            (lambda: backend.attention_mask(torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, 4)), "prefix is"),
            (lambda: backend.attention_mask(torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, 5, dtype=torch.bool)), "prefix must be"),
            (lambda: backend.attention_mask(torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, 4, dtype=torch.bool, device="meta")), "is on meta")):
        with pytest.raises(TrainingError, match=message):
            call()
    mask = backend.AttentionMask(2, 4, torch.zeros(16, dtype=torch.uint8))
    q, k = torch.zeros(4, 8, 64), torch.zeros(4, 4, 64)
    for args, message in (((q, k, k, 3), "do not fit groups"), ((q, k, k[:3], 2), "do not fit"), ((q, k, k.bfloat16(), 2), "q, k and v are"),
                          ((q[0], k, k, 2), "expected"), ((q, k, k, 0), "do not fit")):
        with pytest.raises(TrainingError, match=message):
            backend.attention_masked_forward(*args, 0.1, mask)
    with pytest.raises(TrainingError, match="must come from"):
        backend.attention_masked_forward(q, k, k, 2, 0.1, None)
    for other in (backend.AttentionMask(3, 4, mask.block), backend.AttentionMask(2, 5, mask.block)):
        with pytest.raises(TrainingError, match="does not fit"):
            backend.attention_masked_forward(q, k, k, 2, 0.1, other)
    with pytest.raises(InvalidConfig, match="no gradients"):
        training.grad_norm([])
    for limit in (-1.0, math.nan):
        with pytest.raises(InvalidConfig, match="max_norm"):
            training.AdamW().step_vars([meta], [meta], max_grad_norm=limit)
