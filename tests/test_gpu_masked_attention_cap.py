"""The score cap alone: in documents of one token the log-sum-exp is the score, cap tanh(s / cap)."""
import math

import pytest
import torch

from metal_candle_b200 import backend
from tests.test_gpu_masked_attention import mask_of

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.parametrize("cap", [1.0, 30.0])
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F32, 64)])
def test_capped_scores(cuda_device, dtype, d, cap):
    """q has x in one place and k a one, so that the product is x, exactly.  Where all of a tile lie within the cap, the polynomial: 1.6e-7 of the value and the
    three products behind it (cap log2 e, its constant's rounding, ln 2), 2^-24 each and twice where a constant is rounded.  Beyond, 1 - 2 / (1 + e^2x): the
    exponential to 2^-22 + 2 |x| 2^-24 for its argument's rounding, sum and reciprocal to 2^-23 each, of a quotient that is at most 1, twice that; and the
    last difference."""
    S = 4096
    x = torch.cat([torch.linspace(-1, 1, 1024), torch.linspace(-3, 3, 1024), torch.linspace(-12, 12, 1024), torch.logspace(-8, 3, 1024)]).to(BF16).float()
    q, k = torch.zeros(1, S, d, device=cuda_device), torch.zeros(1, S, d, device=cuda_device)
    q[0, :, 3], k[0, :, 3] = x.to(cuda_device), 1.0
    q, k = q.to(dtype), k.to(dtype)
    mask = mask_of(cuda_device, [list(range(S))], None)
    # the scale of 1 / cap takes x to x / cap, so that the cap bends at |x| = 1 whatever it is
    o, lse = backend.attention_masked_forward(q, k, k, 1, cap, mask, softcap=cap)
    got = lse[0].cpu().double() / cap
    x = x.double()
    want = torch.tanh(x)
    near = 1.6e-7 + 8 * 2.0 ** -24
    far = 2 * (2.0 ** -22 + 2 * x.abs().clamp_max(10) * 2.0 ** -24 + 2 * 2.0 ** -23) + 8 * 2.0 ** -24
    limit = torch.full_like(x, 0.0)
    for at in range(0, S, 32):   # a warp's rows go one way or the other together
        part = slice(at, at + 32)
        limit[part] = near * want[part].abs() if float(x[part].abs().max()) <= 1 else far[part]
    assert ((got - want).abs() <= limit + 1e-45).all(), float(((got - want).abs() - limit).max())
    assert torch.equal(o, k)
