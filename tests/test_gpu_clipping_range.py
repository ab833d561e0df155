"""Clipping by the global norm at the ends of float32, and the norm in a step's metrics."""
import math

import pytest
import torch

from metal_candle_b200 import _lib, training
from metal_candle_b200.training import AdamW, AdamWConfig, clip_grad_norm, grad_norm
from tests.test_gpu_packed_training import rand

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def test_clipping_where_the_norm_passes_float32(cuda_device):
    """Finite gradients whose norm is above 3.4e38: the norm reads inf, and they are scaled to max_norm all the same."""
    for dtype in (F32, BF16):
        for n in (2, 5000):
            g = torch.full((n,), 3e38, device=cuda_device).to(dtype)
            g[1] = -1e38
            whole = math.sqrt(float(g.double().square().sum()))
            for limit in (1.0, 1e-3, 1e30):
                clipped = [g.clone()]
                norm = float(clip_grad_norm(clipped, limit))
                assert norm == math.inf if whole > 3.41e38 else abs(norm - whole) <= 2.0 ** -19 * whole
                want = g.double() * (limit / whole)
                # 16 float32 additions at most in the norm, the factor's and the products' roundings, the output's
                assert ((clipped[0].double() - want).abs() <= (2.0 ** -19 + torch.finfo(dtype).eps / 2) * want.abs()).all()


@pytest.mark.parametrize("size,grad_scale", [(3e38, 2.0 ** -100), (3e38, 1e-30), (1e-40, 2.0 ** 100), (1e38, 1.0)])
def test_adamw_clips_by_the_norm_of_the_scaled_gradients(cuda_device, size, grad_scale):
    """The norm counts after grad_scale, wherever in float32 the gradients lie before it."""
    n, limit = 1000, 0.5
    g = rand(cuda_device, n, seed=1).clamp(-1, 1) * size
    p, a = torch.zeros(n, device=cuda_device), AdamW(AdamWConfig(learning_rate=1e-2, beta1=0.5, beta2=0.5, weight_decay=0.0))
    norm = a.step_vars([p], [g], grad_scale=grad_scale, max_grad_norm=limit)
    scale = float(torch.tensor(grad_scale, dtype=F32))
    whole = math.sqrt(float((g.double() * scale).square().sum()))
    assert abs(float(norm) - whole) <= 2.0 ** -19 * whole if whole < 3.4e38 else float(norm) == math.inf
    want = g.double() * scale * min(1.0, limit / (whole + 1e-6))
    m = a.state_of(p)[0].double()   # (1 - beta1) of the gradient that the update has seen, exactly
    # the norm's 16 additions, the factor, two products; a gradient below 2^-126 before it is scaled has lost digits already
    assert ((2 * m - want).abs() <= 2.0 ** -18 * want.abs() + 1e-44).all() and float(m.abs().max()) > 0


def test_the_norm_reaches_the_metrics(cuda_device):
    params = [rand(cuda_device, 5, seed=1), rand(cuda_device, 7, seed=2)]

    class Adapter:
        def layers(self):
            return [("layers.0.q_proj", self)]

        def trainable_variables(self):
            return params

    grads = [rand(cuda_device, 5, seed=3), rand(cuda_device, 7, seed=4)]
    step = lambda **how: training.TrainingStep().execute(None, None, Adapter(), AdamW(), 1e-3, lambda i, t: (1.0, grads), **how)  # noqa: E731
    assert step().grad_norm is None
    assert step(max_grad_norm=1e-3).grad_norm == float(grad_norm(grads))


@pytest.mark.parametrize("limit", [None, 0.5])
def test_adamw_on_another_device_than_the_current_one(cuda_device, monkeypatch, limit):
    """The update is launched with the parameters' device as the current one (seen here by a current device that is only said to be another)."""
    p, g = rand(cuda_device, 40, seed=1), rand(cuda_device, 40, seed=2)
    other, made = p.clone(), []
    AdamW().step_vars([p], [g], max_grad_norm=limit)
    now = [cuda_device.index + 1]

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index

        def __enter__(self):
            made.append(self.index)
            self.before, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.before

    a = AdamW()
    a.add_parameter(a._key(other), other)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    a.step_vars([other], [g], max_grad_norm=limit)
    monkeypatch.undo()
    assert made and set(made) == {cuda_device.index} and torch.equal(p, other)


@pytest.mark.parametrize("which", range(4))
def test_adamw_refuses_pointers_off_their_elements(cuda_device, which):
    t = [torch.zeros(8, device=cuda_device) for _ in range(4)]
    at = [x.data_ptr() for x in t]
    at[which] += 2
    table = (_lib.AdamWTensor * 1)(_lib.AdamWTensor(*at, 4, 1, 0))
    lib = _lib.init(cuda_device.index)
    assert lib.mcb_adamw_multi(table, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None) == -3
    torch.cuda.synchronize()
    assert not any(x.any() for x in t)
