"""More of what the entry points of training on packed documents refuse, on the CPU: nothing is launched, no pointer is followed."""
import ctypes as C

import pytest
import torch

from metal_candle_b200 import _lib, backend
from metal_candle_b200.backend import TrainingError

NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE, NOT_INIT = -1, -2, -3, -4, -5, -6
F32, BF16 = _lib.MCB_F32, _lib.MCB_BF16
HUGE = 1 << 40
FAR = [(i + 2) << 41 for i in range(12)]


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def each(call, count, good, bad, dtype):
    """call(pointers) reaches the device with pointers far apart, and refuses each of the first `count` off its boundary."""
    args = list(FAR[:count])
    assert call(args) == NOT_INIT
    for i in range(count):
        for off in (good[i], bad[i]):
            args = list(FAR[:count])
            args[i] += off
            assert call(args) == (NOT_INIT if off == good[i] else ALIGN), (i, off, dtype)


@pytest.mark.parametrize("dtype,size", [(F32, 4), (BF16, 2)])
def test_pointers_off_their_elements(lib, dtype, size):
    """A load of an element off its boundary would fault the device: refused.  On the boundary of an element every call goes on."""
    part = size // 2
    each(lambda p: lib.mcb_layernorm_fwd(p[0], p[1], p[2], p[3], p[4], p[5], 4, 8, 1e-5, dtype, None), 6, [size] * 4 + [4] * 2, [part] * 4 + [2] * 2, dtype)
    each(lambda p: lib.mcb_layernorm_bwd(p[0], p[1], p[2], p[3], p[4], p[5], p[6], 0, 4, 8, 1e-5, dtype, 16, HUGE, None), 7, [size] * 5 + [4] * 2,
         [part] * 5 + [2] * 2, dtype)
    for id_bytes in (4, 8):
        each(lambda p: lib.mcb_embedding_scaled_fwd(p[0], id_bytes, p[1], p[2], 4, 8, 10, 1.0, dtype, None), 3, [id_bytes, size, size],
             [id_bytes // 2, part, part], dtype)
        each(lambda p: lib.mcb_embedding_bwd(p[0], id_bytes, p[1], FAR[5], 0, 4, 8, 10, 1.0, dtype, 16, HUGE, None), 2, [id_bytes, size], [id_bytes // 2, part],
             dtype)


def test_statistics_off_their_elements(lib):
    call = _lib.MaskedAttention(16, HUGE, None, 2, 100, 2, 3, 64, 0.125, 0.0, BF16, 0)
    f = FAR
    for off, status in ((4, NOT_INIT), (2, ALIGN)):
        assert lib.mcb_attention_masked_fwd(C.byref(call), f[0], f[1], f[2], f[3], f[4] + off, None) == status
        assert lib.mcb_attention_masked_bwd(C.byref(call), f[0], f[1], f[2], f[3], f[4] + off, f[5], f[6], f[7], f[8], 1 << 50, HUGE, None) == status
        grads = (_lib.GradTensor * 1)(_lib.GradTensor(f[0], None, 10, F32, 0))
        assert lib.mcb_grad_norm(grads, 1, f[1] + off, 16, HUGE, None) == status
        assert lib.mcb_clip_grad_norm(grads, 1, 1.0, f[1] + off, 16, HUGE, None) == status
        table = (_lib.AdamWTensor * 1)(_lib.AdamWTensor(f[0], f[1], f[2], f[3], 4, 1, 0))
        assert lib.mcb_adamw_multi_clipped(table, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 1.0, f[4] + off, 16, HUGE, None) == status


def test_layer_norm_outputs_overlap_nothing_else(lib):
    rows, D = 4, 8
    all_, row, stat = rows * D * 4, D * 4, rows * 4
    f = FAR
    fwd = lambda p: lib.mcb_layernorm_fwd(p[0], p[1], p[2], p[3], p[4], p[5], rows, D, 1e-5, F32, None)  # noqa: E731
    sizes = [all_, row, row, all_, stat, stat]   # x, w, b, y, mean, rstd
    for out in (3, 4, 5):
        for i in range(6):
            if i == out:
                continue
            for at, status in ((f[i], NOT_INIT if (out, i) == (3, 0) else SHAPE), (f[i] + sizes[i] - 4, SHAPE), (f[i] + sizes[i], NOT_INIT),
                               (f[i] - sizes[out] + 4, SHAPE), (f[i] - sizes[out], NOT_INIT)):
                args = f[:6]
                args[out] = at
                assert fwd(args) == status, (out, i, at - f[i])
    ws = lib.mcb_layernorm_bwd_workspace_bytes(rows, D)
    bwd = lambda p: lib.mcb_layernorm_bwd(p[0], p[1], p[2], p[3], p[4], p[5], p[6], 0, rows, D, 1e-5, F32, p[7], HUGE, None)  # noqa: E731
    sizes = [all_, row, all_, all_, all_, row, row, ws]   # x, w, dy, dx_residual, dx, dw, db, workspace
    for out in (4, 5, 6, 7):
        for i in range(8):
            if i == out:
                continue
            for at, status in ((f[i], NOT_INIT if out == 4 and i in (0, 2, 3) else SHAPE), (f[i] + sizes[i] - 16, SHAPE), (f[i] + sizes[i], NOT_INIT),
                               (f[i] - sizes[out] + 16, SHAPE), (f[i] - sizes[out], NOT_INIT)):
                args = f[:8]
                args[out] = at
                assert bwd(args) == status, (out, i, at - f[i])
    both = f[:8]
    both[2] = both[3] = both[4] = f[0]
    assert bwd(both) == NOT_INIT
    alone = list(f[:8])
    alone[5], alone[6], alone[7] = None, None, f[0]   # no sums: the workspace is not used
    assert bwd(alone) == NOT_INIT


def test_embedding_outputs_overlap_nothing(lib):
    M, H, V, f = 4, 8, 10, FAR
    for id_bytes in (4, 8):
        fwd = lambda ids, table, out: lib.mcb_embedding_scaled_fwd(ids, id_bytes, table, out, M, H, V, 1.0, BF16, None)  # noqa: E731
        assert fwd(f[0], f[1], f[1] + 2 * V * H) == NOT_INIT and fwd(f[0], f[1], f[1] + 2 * V * H - 2) == SHAPE
        assert fwd(f[0], f[1], f[1] - 2 * M * H) == NOT_INIT and fwd(f[0], f[1], f[1]) == SHAPE
        assert fwd(f[0], f[1], f[0] + id_bytes * M) == NOT_INIT and fwd(f[0], f[1], f[0] + id_bytes * M - 2) == SHAPE
        bwd = lambda ids, dout, grad, ws: lib.mcb_embedding_bwd(ids, id_bytes, dout, grad, 0, M, H, V, 1.0, F32, ws, HUGE, None)  # noqa: E731
        need = lib.mcb_embedding_bwd_workspace_bytes(M, H)
        assert bwd(f[0], f[1], f[2], f[3]) == NOT_INIT
        for other, size in ((f[0], id_bytes * M), (f[1], 4 * M * H)):
            assert bwd(f[0], f[1], other, f[3]) == SHAPE and bwd(f[0], f[1], other + size - 16, f[3]) == SHAPE and bwd(f[0], f[1], other + size, f[3]) == NOT_INIT
            assert bwd(f[0], f[1], f[2], other - need + 16) == SHAPE and bwd(f[0], f[1], f[2], other - need) == NOT_INIT
        assert bwd(f[0], f[1], f[2], f[2] + 4 * V * H - 16) == SHAPE and bwd(f[0], f[1], f[2], f[2] + 4 * V * H) == NOT_INIT


def test_attention_outputs_do_not_overlap_the_slopes(lib):
    call = _lib.MaskedAttention(16, HUGE, FAR[9], 2, 100, 2, 3, 64, 0.125, 0.0, BF16, 0)
    f = FAR
    assert lib.mcb_attention_masked_fwd(C.byref(call), *f[:5], None) == NOT_INIT
    for i in (3, 4):
        args = f[:5]
        args[i] = f[9] + 16
        assert lib.mcb_attention_masked_fwd(C.byref(call), *args, None) == SHAPE
    for i in (6, 7, 8):
        args = f[:9]
        args[i] = f[9] + 16
        assert lib.mcb_attention_masked_bwd(C.byref(call), *args, 1 << 50, HUGE, None) == SHAPE
    assert lib.mcb_attention_masked_bwd(C.byref(call), *f[:9], f[9], HUGE, None) == SHAPE
    assert lib.mcb_attention_masked_bwd(C.byref(call), *f[:9], f[9] + 1024, HUGE, None) == NOT_INIT


def test_a_mask_of_other_sizes_than_its_documents():
    ids, marks = torch.zeros(2, 5, dtype=torch.int32, device="meta"), torch.zeros(2, 5, dtype=torch.bool, device="meta")
    for given in (dict(document_ids=ids), dict(prefix=marks), dict(document_ids=ids, prefix=marks)):
        for other, message in ((dict(batch=3), "do not fit"), (dict(seq=4), "do not fit"), (dict(batch=2, seq=10), "do not fit"), (dict(device="cuda"), "but document_ids"),
                               (dict(batch=2, seq=5, device="meta"), "CUDA device"), (dict(), "CUDA device")):
            with pytest.raises(TrainingError, match=message):
                backend.attention_mask(**given, **other)


@pytest.mark.parametrize("batch,seq", [(1, 1), (65535, 1), (2, 4096), (8, 128), (1, 32768), (3, 1000), (1, 32769), (2, 70001)])
def test_bytes_of_a_mask(lib, batch, seq):
    """Four numbers a position, twelve a tile of 128 and, beyond 32768 positions, two bitmaps of three levels, a word for 32 each."""
    tiles, chunks = (seq + 127) // 128, (seq + 32767) // 32768
    words = batch * (4 * seq + 12 * tiles + (2 * chunks * 1057 if seq > 32768 else 0))
    assert 4 * words <= lib.mcb_attention_mask_bytes(batch, seq) <= 4 * words + 48


@pytest.mark.parametrize("scale,softcap,status", [(0.125, 1.7e38, SHAPE), (0.125, 2.0 ** 124, SHAPE), (0.125, 2.0 ** 123, NOT_INIT), (2.0 ** -100, 2.0 ** 27, SHAPE),
                                                  (2.0 ** -100, 2.0 ** 26, NOT_INIT), (1.0, 0.0, NOT_INIT), (1e-38, 0.0, NOT_INIT)])
def test_caps_whose_quotient_has_lost_digits(lib, scale, softcap, status):
    """scale / softcap below 2^-126 is held with fewer digits: the scores would be wrong by as much."""
    call = _lib.MaskedAttention(16, HUGE, None, 2, 100, 2, 3, 64, scale, softcap, F32, 0)
    assert lib.mcb_attention_masked_fwd(C.byref(call), *FAR[:5], None) == status
    assert lib.mcb_attention_masked_bwd(C.byref(call), *FAR[:9], 1 << 50, HUGE, None) == status
