"""Masked attention where values are not finite, over long documents: rows that are taken again by themselves."""
import math

import pytest
import torch

from metal_candle_b200 import backend
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
