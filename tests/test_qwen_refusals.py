"""Tokens on another device than the model's, refused before any kernel gets their address.  On the CPU: the model is a shell whose
weights are on no device at all."""
import pytest
import torch

from metal_candle_b200.backend import TrainingError
from metal_candle_b200.qwen import ModelConfig, Qwen

B, S = 2, 3


@pytest.fixture
def shell():
    model = Qwen.__new__(Qwen)
    model.config = ModelConfig()
    model.dtype, model.device = torch.bfloat16, torch.device("meta")
    model.embed_tokens = torch.empty(8, 4, device="meta")
    model.lora_adapter = object()
    model.fuse_swiglu_bwd = True
    model.layers = []
    return model


def on(device, dtype=torch.int64, *shape):
    return torch.zeros(shape or (B, S), dtype=dtype, device=device)


IDS = {
    "forward": lambda m, i: m.forward(i),
    "forward_backward": lambda m, i: m.forward_backward(i, on("meta")),
    "token_log_probs": lambda m, i: m.token_log_probs(i, on("meta")),
    "preference": lambda m, i: m.preference_forward_backward(i, on("meta"), on("meta", torch.float32, B)),
    "policy": lambda m, i: m.policy_forward_backward(i, on("meta"), on("meta", torch.float32, B)),
    "distillation": lambda m, i: m.distillation_forward_backward(i, on("meta", torch.int64, B, S, 1), on("meta", torch.float32, B, S, 1)),
}


@pytest.mark.parametrize("call", IDS)
def test_input_ids_on_the_host(shell, call):
    with pytest.raises(TrainingError, match="input_ids is on cpu"):
        IDS[call](shell, on("cpu"))


def test_targets_on_the_host(shell):
    for f in (lambda: shell.forward_backward(on("meta"), on("cpu")), lambda: shell.token_log_probs(on("meta"), on("cpu"))):
        with pytest.raises(TrainingError, match="target_ids is on cpu"):
            f()
