"""GPU: post-training passes of the model -- scoring, preference, policy and distillation steps -- whose logits exist a chunk of
tokens at a time, against the losses over whole logits and against the cross-entropy step they come down to."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

B, S, V = 4, 24, 320


def small_model(dev, dtype, seed=5):
    from metal_candle_b200.qwen import ModelConfig, Qwen
    from metal_candle_b200.training import LoRAAdapter, LoRAAdapterConfig, TargetModule

    cfg = ModelConfig(vocab_size=V, hidden_size=256, intermediate_size=384, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      max_position_embeddings=256)
    model = Qwen(cfg, dev, dtype=dtype, seed=seed)
    g = torch.Generator(device=dev).manual_seed(6)
    acfg = LoRAAdapterConfig(rank=8, alpha=16.0, target_modules=[TargetModule.QProj, TargetModule.KProj, TargetModule.VProj, TargetModule.OProj])
    adapter = LoRAAdapter(cfg.hidden_size, cfg.intermediate_size, cfg.num_hidden_layers, acfg, dev, kv_size=cfg.kv_size, generator=g)
    for _, l in adapter.layers():
        l.lora_a.mul_(0.3)
        l.lora_b.normal_(0, 0.05, generator=g)
    model.apply_adapter(adapter)
    ids = torch.randint(0, V, (B, S), device=dev, generator=g)
    targets = torch.cat([ids[:, 1:], torch.full((B, 1), -1, device=dev)], 1)
    targets[:, :5] = -1
    return model, ids, targets, g


def close(a, b, rel):
    """Of the largest element."""
    for u, v in zip(a, b):
        assert (u - v).abs().max() <= rel * max(float(v.abs().max()), 1e-12), (float((u - v).abs().max()), float(v.abs().max()))


def clones(grads):
    return [g.clone() for g in grads]


# float32: sums of 1e-6 through two layers; bfloat16: a gradient of the logits is rounded to 2^-8 of itself, and those roundings
# and the ones behind them (some ten a layer) average out over the sums to a few of them
REL = {torch.float32: 1e-4, torch.bfloat16: 4e-2}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_losses_that_come_down_to_cross_entropy(cuda_device, dtype):
    """With r = 1 and advantage 1 the policy loss has the gradient of cross-entropy; distillation from one entry is cross-entropy."""
    model, ids, targets, g = small_model(cuda_device, dtype)
    loss, grads = model.forward_backward(ids, targets)
    want = clones(grads)
    out, grads = model.policy_forward_backward(ids, targets, torch.ones(B, device=cuda_device))
    assert abs(float(out.loss) + 1) < 1e-6
    close(grads, want, REL[dtype])
    kept = targets >= 0
    assert abs(-float(out.log_probs[kept].mean()) - float(loss)) < 1e-2 * float(loss)
    dl, grads = model.distillation_forward_backward(ids, targets.clamp_min(0)[..., None], torch.zeros(B, S, 1, device=cuda_device), mask=kept)
    assert abs(float(dl) - float(loss)) < 1e-2 * float(loss)
    close(grads, want, REL[dtype])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_chunks_and_whole_logits_agree(cuda_device, dtype):
    from metal_candle_b200 import training as F

    model, ids, targets, g = small_model(cuda_device, dtype)
    with model.adapter_disabled():
        ref = model.token_log_probs(ids, targets)
        base = model.forward(ids)
    logits = model.forward(ids)
    assert not torch.equal(base, logits) and model.layers[0]["q_proj"].lora is not None
    torch.testing.assert_close(ref, F.token_log_probs(base, targets)[0], rtol=1e-5, atol=1e-5)
    old = model.token_log_probs(ids, targets, temperature=0.8) + 0.1 * torch.randn(B, S, device=cuda_device, generator=g)
    adv = torch.randn(B, device=cuda_device, generator=g)
    tids = torch.topk(base.float(), 16, dim=-1).indices
    tl = base.gather(-1, tids)
    opts = dict(kl_coef=0.1, temperature=0.8, sequence_mean=True)
    whole = (F.policy_loss(logits, targets, adv, old, ref, **opts), F.preference_loss(logits, targets, ref.sum(1)),
             F.distillation_loss(logits, tids, tl, mask=targets >= 0, temperature=2.0))
    first = None
    for chunk in (None, 96, 40, 7):   # one, one, and chunks that begin and end inside sequences
        model.ce_chunk_tokens = chunk
        pol, grads = model.policy_forward_backward(ids, targets, adv, old, ref, **opts)
        got = [clones(grads)]
        pref, grads = model.preference_forward_backward(ids, targets, ref.sum(1))
        got.append(clones(grads))
        dist, grads = model.distillation_forward_backward(ids, tids, tl, mask=targets >= 0, temperature=2.0)
        got.append(clones(grads))
        # the lm_head of a chunk may take another kernel, whose sums differ in order: 1e-5 in float32, a rounding of the
        # logits (2^-8 of at most 2 or so, and averaged) in bfloat16
        tol = 1e-4 if dtype == torch.float32 else 2e-2
        assert abs(float(pol.loss) - float(whole[0].loss)) < tol and abs(float(pol.kl) - float(whole[0].kl)) < tol
        assert (pol.log_probs - whole[0].log_probs).abs().max() < tol
        assert abs(float(pref.loss) - float(whole[1].loss)) < tol
        assert (pref.log_probs - whole[1].log_probs).abs().max() < S * tol
        assert abs(float(dist) - float(whole[2])) < tol
        if first is None:
            first = got
        for a, b in zip(got, first):
            close(a, b, REL[dtype])
    # accumulate adds to what is there
    model.ce_chunk_tokens = 40
    _, grads = model.policy_forward_backward(ids, targets, adv, old, ref, **opts)
    one = clones(grads)
    _, grads = model.policy_forward_backward(ids, targets, adv, old, ref, accumulate=True, **opts)
    close(grads, [2 * v for v in one], 1e-5)


def test_adapter_gradients_against_differences(cuda_device):
    """float32: d loss along a direction of the adapters' parameters against the loss's difference quotient.  The loss is good to some
    1e-6; h = 0.01 along a direction of unit length makes that 1e-4 of noise, and as much again of curvature."""
    model, ids, targets, g = small_model(cuda_device, torch.float32)
    variables = [v for _, l in model.lora_adapter.layers() for v in l.trainable_variables()]
    with model.adapter_disabled():
        ref = model.token_log_probs(ids, targets)
        base = model.forward(ids)
    old = model.token_log_probs(ids, targets) + 0.05
    adv = torch.randn(B, device=cuda_device, generator=g)
    tids = torch.topk(base + torch.randn(base.shape, device=cuda_device, generator=g), 8, dim=-1).indices
    tl = torch.randn(B, S, 8, device=cuda_device, generator=g)
    passes = {
        "policy": lambda: model.policy_forward_backward(ids, targets, adv, old, ref, kl_coef=0.5, clip_low=0.9, clip_high=5.0),
        "preference": lambda: model.preference_forward_backward(ids, targets, ref.sum(1), beta=0.2),
        "distill": lambda: model.distillation_forward_backward(ids, tids, tl, temperature=1.3),
    }
    value = lambda out: float(out[0].loss if hasattr(out[0], "loss") else out[0])  # noqa: E731
    for name, f in passes.items():
        _, grads = f()
        grads = clones(grads)
        norm = math.sqrt(sum(float(v.double().pow(2).sum()) for v in grads))
        h, quotient = 0.01, 0.0
        for sign in (1, -1):
            for v, d in zip(variables, grads):
                v.add_(d, alpha=sign * h / norm)
            quotient += sign * value(f()) / (2 * h)
            for v, d in zip(variables, grads):
                v.add_(d, alpha=-sign * h / norm)
        assert norm > 1e-3 and abs(quotient - norm) <= 1e-2 * norm + 2e-4, (name, quotient, norm)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_run_of_post_training_steps(cuda_device, dtype):
    """Scoring with the frozen base, then preference, policy and distillation steps with the optimizer, and a graph of one of them
    replayed while eager passes run between: same gradients."""
    from metal_candle_b200.training import AdamW, AdamWConfig, TrainingStep

    model, ids, targets, g = small_model(cuda_device, dtype)
    opt, step = AdamW(AdamWConfig()), TrainingStep()
    with model.adapter_disabled():
        ref = model.token_log_probs(ids, targets)
    adv = torch.randn(B, device=cuda_device, generator=g)
    old = model.token_log_probs(ids, targets)

    def policy(i, t):
        out, grads = model.policy_forward_backward(i, t, adv, old, ref, kl_coef=0.04)
        return out.loss, grads

    def preference(i, t):
        out, grads = model.preference_forward_backward(i, t, ref.sum(1))
        return out.loss, grads

    tids = torch.topk(model.forward(ids).float(), 8, dim=-1)
    before = [l.lora_b.clone() for _, l in model.lora_adapter.layers()]
    for fn in (policy, preference, lambda i, t: model.distillation_forward_backward(i, tids.indices, tids.values.to(dtype), mask=t >= 0)):
        m = step.execute(ids, targets, model.lora_adapter, opt, 1e-4, fn)
        assert math.isfinite(m.loss)
    assert all(not torch.equal(a, l.lora_b) for a, (_, l) in zip(before, model.lora_adapter.layers()))

    _, grads = policy(ids, targets)
    want = clones(grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = policy(ids, targets)
    for _ in range(2):
        preference(ids, targets)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_model_passes_refuse(cuda_device):
    from metal_candle_b200.backend import TrainingError

    model, ids, targets, g = small_model(cuda_device, torch.bfloat16)
    one = torch.ones(B, device=cuda_device)
    with pytest.raises(TrainingError, match="pairs"):
        model.preference_forward_backward(ids[:3], targets[:3], one[:3])
    with pytest.raises(TrainingError, match="target_ids"):
        model.policy_forward_backward(ids, targets[:, :-1], one)
    with pytest.raises(TrainingError, match="advantages"):
        model.policy_forward_backward(ids, targets, one[:2])
    with pytest.raises(TrainingError, match="temperature"):
        model.token_log_probs(ids, targets, temperature=0.0)
    with pytest.raises(TrainingError, match="teacher_ids"):
        model.distillation_forward_backward(ids, ids, one)
    model.remove_adapter()
    for f in (lambda: model.policy_forward_backward(ids, targets, one), lambda: model.preference_forward_backward(ids, targets, one)):
        with pytest.raises(TrainingError, match="adapter"):
            f()
