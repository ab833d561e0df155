"""More of what the entry points of training on packed documents refuse, on the CPU: nothing is launched, no pointer is followed."""
import ctypes as C

import pytest

from metal_candle_b200 import _lib

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
