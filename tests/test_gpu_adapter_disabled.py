"""GPU: what a model refuses while its adapter is set aside, and that the adapter is back afterwards."""
import pytest
import torch

from tests.test_gpu_post_training import B, clones, small_model

pytestmark = pytest.mark.gpu


def test_training_passes_are_refused(cuda_device):
    from metal_candle_b200.backend import TrainingError
    from metal_candle_b200.engine import QwenEngine

    model, ids, targets, g = small_model(cuda_device, torch.bfloat16)
    one = torch.ones(B, device=cuda_device)
    teacher = torch.zeros(*ids.shape, 1, device=cuda_device)
    _, grads = model.forward_backward(ids, targets)
    want = clones(grads)
    passes = [lambda: model.forward_backward(ids, targets), lambda: model.policy_forward_backward(ids, targets, one),
              lambda: model.preference_forward_backward(ids, targets, one),
              lambda: model.distillation_forward_backward(ids, ids[..., None], teacher),
              lambda: model.capture_forward_backward(*ids.shape), lambda: QwenEngine(model, *ids.shape)]
    with model.adapter_disabled():
        assert not model.has_adapter()
        for f in passes:
            with pytest.raises(TrainingError, match="adapter"):
                f()
        base = model.token_log_probs(ids, targets)
        with model.adapter_disabled():   # one within another
            assert torch.equal(model.token_log_probs(ids, targets), base)
        assert not model.has_adapter()
    assert model.has_adapter()
    assert all(torch.equal(a, b) for a, b in zip(model._grad_views, want))   # nobody has written there
    _, grads = model.forward_backward(ids, targets)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_adapters_are_not_exchanged_meanwhile(cuda_device):
    from metal_candle_b200.backend import TrainingError

    model, ids, targets, g = small_model(cuda_device, torch.float32)
    adapter = model.lora_adapter
    lora = model.layers[0]["q_proj"].lora
    with pytest.raises(RuntimeError, match="on the way"):
        with model.adapter_disabled():
            for f in (lambda: model.apply_adapter(adapter), model.remove_adapter):
                with pytest.raises(TrainingError, match="adapter_disabled"):
                    f()
            raise RuntimeError("on the way")
    assert model.lora_adapter is adapter and model.layers[0]["q_proj"].lora is lora
    model.remove_adapter()
    with model.adapter_disabled():   # nothing to set aside
        model.token_log_probs(ids, targets)
    assert not model.has_adapter()
    model.apply_adapter(adapter)
    assert model.has_adapter()
