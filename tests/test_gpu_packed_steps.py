"""Steps beside the model's passes over packed documents: captured ones, the engine's."""
import pytest
import torch

from metal_candle_b200.backend import TrainingError
from tests.test_gpu_post_training import V, small_model

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_steps_without_documents_are_refused_within_packed(cuda_device):
    """A step captured before, or the engine's, would run the batch as one text."""
    from metal_candle_b200.engine import QwenEngine

    model, _, _, g = small_model(cuda_device, BF16)
    ids = torch.randint(0, V, (2, 128), device=cuda_device, generator=g)   # (the engine takes lengths of 128)
    targets = ids.roll(-1, 1)
    model.forward_backward(ids, targets)
    step = model.capture_forward_backward(*ids.shape)
    engine = QwenEngine(model, *ids.shape)
    ids32, targets32 = ids.to(torch.int32), targets.to(torch.int32)
    loss = step(ids, targets)[0].clone()
    with model.packed(torch.zeros_like(ids)):
        for call in (lambda: step(ids, targets), lambda: engine.forward_backward(ids32, targets32), lambda: engine.train_step(ids32, targets32, 1e-3)):
            with pytest.raises(TrainingError, match="packed"):
                call()
    assert torch.equal(step(ids, targets)[0], loss)
    engine.forward_backward(ids32, targets32)
