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


def test_a_capture_by_hand_holds_its_own_documents(cuda_device):
    """packed() opened while a graph is recorded belongs to it; a block opened before does not, and the graph would outlive it."""
    model, ids, targets, _ = small_model(cuda_device, BF16)
    docs = torch.arange(ids.shape[1], device=cuda_device, dtype=torch.int32).expand(ids.shape).contiguous() // 7
    with model.packed(docs):
        want = model.forward_backward(ids, targets)[0].clone()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(TrainingError, match="packed"):
            with torch.cuda.graph(graph):
                model.forward_backward(ids, targets)
    plain = model.forward_backward(ids, targets)[0].clone()
    graph, held = torch.cuda.CUDAGraph(), docs.clone()
    with torch.cuda.graph(graph):
        with model.packed(held):
            loss, grads = model.forward_backward(ids, targets)
    graph.replay()
    assert torch.equal(loss, want) and not torch.equal(loss, plain)
    held.zero_()   # other documents, the same graph
    graph.replay()
    one = loss.clone()
    with model.packed(torch.zeros_like(docs)):
        assert torch.equal(model.forward_backward(ids, targets)[0], one)
