"""Refusals of the losses over given tokens, on the CPU: nothing reaches a device before its arguments have been checked."""
import ctypes as C
import math

import pytest
import torch

from metal_candle_b200 import _lib
from metal_candle_b200 import training as F
from metal_candle_b200.backend import TrainingError

B, S, V, K = 4, 3, 7, 2


def good(**change):
    args = dict(logits=torch.zeros(B, S, V), targets=torch.zeros(B, S, dtype=torch.int64), ref=torch.zeros(B), adv=torch.zeros(B),
                ids=torch.zeros(B, S, K, dtype=torch.int64), teacher=torch.zeros(B, S, K), tok=torch.zeros(B, S))
    args.update(change)
    return args


CALLS = {
    "log_probs": lambda a, **k: F.token_log_probs(a["logits"], a["targets"], **k),
    "backward": lambda a, **k: F.token_log_probs_backward(a["logits"], a["targets"], a["tok"], a["tok"], a["tok"], **k),
    "preference": lambda a, **k: F.preference_loss(a["logits"], a["targets"], a["ref"], **k),
    "policy": lambda a, **k: F.policy_loss(a["logits"], a["targets"], a["adv"], **k),
    "distill": lambda a, **k: F.distillation_loss(a["logits"], a["ids"], a["teacher"], **k),
}


@pytest.mark.parametrize("call", CALLS)
def test_no_cpu_path(call):
    with pytest.raises(TrainingError, match="no CPU path"):
        CALLS[call](good())


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("change,what", [
    (dict(logits=torch.zeros(S, V)), "3D"),
    (dict(logits=torch.zeros(B, S, 0)), "empty"),
    (dict(logits=torch.zeros(B, S, V, dtype=torch.float16)), "unsupported dtype"),
])
def test_logits_refused(call, change, what):
    with pytest.raises(TrainingError, match=what):
        CALLS[call](good(**change))


@pytest.mark.parametrize("call", ["log_probs", "backward", "preference", "policy"])
@pytest.mark.parametrize("targets", [torch.zeros(B, S + 1, dtype=torch.int64), torch.zeros(B * S, dtype=torch.int64), torch.zeros(B, S),
                                     torch.zeros(B, S, dtype=torch.int16)])
def test_targets_refused(call, targets):
    with pytest.raises(TrainingError, match="targets"):
        CALLS[call](good(targets=targets))


@pytest.mark.parametrize("call", ["log_probs", "backward", "policy", "distill"])
@pytest.mark.parametrize("temperature", [0.0, -1.0, math.inf, math.nan, 1e-9])
def test_temperature_refused(call, temperature):
    with pytest.raises(F.InvalidConfig, match="temperature"):
        CALLS[call](good(), temperature=temperature)


@pytest.mark.parametrize("call,change,options,what", [
    ("preference", dict(logits=torch.zeros(3, S, V)), {}, "pairs"),
    ("preference", dict(ref=torch.zeros(B, S)), {}, "ref_log_probs"),
    ("preference", dict(ref=torch.zeros(B, dtype=torch.float64)), {}, "ref_log_probs"),
    ("preference", {}, dict(beta=0.0), "beta"),
    ("preference", {}, dict(beta=math.nan), "beta"),
    ("preference", {}, dict(label_smoothing=-0.1), "label_smoothing"),
    ("preference", {}, dict(label_smoothing=0.6), "label_smoothing"),
    ("policy", dict(adv=torch.zeros(S)), {}, "advantages"),
    ("policy", dict(adv=torch.zeros(B, S + 1)), {}, "advantages"),
    ("policy", dict(adv=torch.zeros(B, dtype=torch.bfloat16)), {}, "advantages"),
    ("policy", {}, dict(old_log_probs=torch.zeros(B)), "old_log_probs"),
    ("policy", {}, dict(ref_log_probs=torch.zeros(B, S, dtype=torch.float64)), "ref_log_probs"),
    ("policy", {}, dict(kl_coef=0.1), "KL"),
    ("policy", {}, dict(kl_coef=-0.1, ref_log_probs=torch.zeros(B, S)), "kl_coef"),
    ("policy", {}, dict(kl_coef=math.inf, ref_log_probs=torch.zeros(B, S)), "kl_coef"),
    ("policy", {}, dict(clip_low=-0.1), "clip"),
    ("policy", {}, dict(clip_high=math.nan), "clip"),
    ("distill", dict(ids=torch.zeros(B, S, dtype=torch.int64)), {}, "teacher_ids"),
    ("distill", dict(ids=torch.zeros(B, S, 0, dtype=torch.int64)), {}, "teacher_ids"),
    ("distill", dict(ids=torch.zeros(B, S, 1025, dtype=torch.int64)), {}, "teacher_ids"),
    ("distill", dict(ids=torch.zeros(B, S, K)), {}, "teacher_ids"),
    ("distill", dict(teacher=torch.zeros(B, S, K + 1)), {}, "teacher_logits"),
    ("distill", dict(teacher=torch.zeros(B, S, K, dtype=torch.float16)), {}, "teacher_logits"),
    ("distill", {}, dict(mask=torch.ones(B, S)), "mask"),
    ("distill", {}, dict(mask=torch.ones(B, dtype=torch.bool)), "mask"),
    ("backward", dict(tok=torch.zeros(B, S, dtype=torch.float64)), {}, "log_probs"),
])
def test_arguments_refused(call, change, options, what):
    with pytest.raises(TrainingError, match=what):
        CALLS[call](good(**change), **options)


def rows(**change):
    """A descriptor no call may get past: the addresses are only looked at for alignment."""
    f = dict(logits=16, batch=2, seq=3, vocab=8, batch_stride=24, token_stride=8, temperature=1.0, dtype=_lib.MCB_F32)
    f.update(change)
    return _lib.TokenLogits(**f)


def targets(**change):
    f = dict(targets=16, target_bytes=8, has_ignore=0, ignore_index=0)
    f.update(change)
    return _lib.TokenTargets(**f)


NULL, SHAPE, ALIGN, UNSUPPORTED, WORKSPACE = -1, -2, -3, -4, -5


def test_c_vocabularies_that_32_bits_do_not_hold():
    lib = _lib.load()
    r = C.byref(rows(vocab=(1 << 30) + 1))
    assert lib.mcb_token_logprob_fwd(r, C.byref(targets()), 16, None, None, None) == SHAPE


@pytest.mark.parametrize("grad", [1024 + 4, 1024 - 4, 1024 + 4 * 47, 1024 - 4 * 47])
def test_c_gradients_that_overlap_in_part(grad):
    lib = _lib.load()
    r = C.byref(rows(logits=1024))
    assert lib.mcb_token_logprob_fwd(r, C.byref(targets()), 16, None, grad, None) == SHAPE
    assert lib.mcb_token_logprob_bwd(r, C.byref(targets()), 16, 16, 16, 1, grad, None) == SHAPE
    assert b"overlaps" in lib.mcb_last_error()
    # a wide stride between sequences, the gradient in the gap
    r = C.byref(rows(logits=1024, batch_stride=1 << 40))
    assert lib.mcb_token_logprob_fwd(r, C.byref(targets()), 16, None, 1024 + 4096, None) == SHAPE


@pytest.mark.parametrize("change,code", [
    (dict(logits=0), NULL), (dict(batch=0), SHAPE), (dict(seq=-1), SHAPE), (dict(vocab=0), SHAPE), (dict(vocab=1 << 31), SHAPE),
    (dict(batch=1 << 20, seq=1 << 20), SHAPE), (dict(batch=1 << 62, seq=4), SHAPE), (dict(batch_stride=-1), SHAPE), (dict(token_stride=-8), SHAPE),
    (dict(temperature=0.0), SHAPE), (dict(temperature=math.nan), SHAPE), (dict(temperature=math.inf), SHAPE), (dict(temperature=1e-39), SHAPE),
    (dict(dtype=2), UNSUPPORTED), (dict(logits=18), ALIGN),
])
def test_c_logits_refused(change, code):
    lib = _lib.load()
    r, t = C.byref(rows(**change)), C.byref(targets())
    pol = C.byref(_lib.PolicyTerms(16, 1, None, None, 0.2, 0.2, 0.0, 0))
    top = C.byref(_lib.TeacherTop(16, 16, 2, 8, 0))
    ws = 1 << 40
    assert lib.mcb_token_logprob_fwd(r, t, 16, 16, None, None) == code
    assert lib.mcb_token_logprob_bwd(r, t, 16, 16, 16, 1, 16, None) == code
    assert lib.mcb_preference_loss(r, t, 16, 0.1, 0.0, 0, 16, 16, None, 16, ws, None) == code
    assert lib.mcb_policy_loss(r, t, pol, 0, 16, 16, None, 16, ws, None) == code
    assert lib.mcb_policy_loss_rows(r, t, pol, 16, 16, 16, None, None) == code
    assert lib.mcb_distill_loss(r, top, None, 16, None, 16, ws, None) == code
    assert lib.mcb_distill_loss_rows(r, top, 16, 16, None, None) == code


def test_c_arguments_refused():
    lib = _lib.load()
    r, t = C.byref(rows()), C.byref(targets())
    ws = 1 << 40
    one = C.byref(_lib.PolicyTerms(16, 1, None, None, 0.2, 0.2, 0.0, 0))
    assert lib.mcb_policy_loss(r, t, one, 0, 16, 16, None, 24, ws, None) == ALIGN
    assert lib.mcb_token_logprob_fwd(None, t, 16, 16, None, None) == NULL
    assert lib.mcb_token_logprob_fwd(r, None, 16, 16, None, None) == NULL
    assert lib.mcb_token_logprob_fwd(r, C.byref(targets(targets=0)), 16, 16, None, None) == NULL
    assert lib.mcb_token_logprob_fwd(r, C.byref(targets(target_bytes=2)), 16, 16, None, None) == UNSUPPORTED
    assert lib.mcb_token_logprob_fwd(r, t, None, 16, None, None) == NULL
    assert lib.mcb_token_logprob_fwd(C.byref(rows(token_stride=9, batch_stride=27)), t, 16, 16, 16, None) == SHAPE   # in place, not dense
    assert lib.mcb_token_logprob_fwd(r, t, 16, 16, 18, None) == ALIGN
    assert lib.mcb_token_logprob_bwd(r, t, 16, 16, 16, 0, 32, None) == SHAPE
    assert lib.mcb_token_logprob_bwd(r, t, 16, None, 16, 1, 32, None) == NULL
    assert lib.mcb_preference_loss(C.byref(rows(batch=3)), t, 16, 0.1, 0.0, 0, 16, 16, None, 16, ws, None) == SHAPE
    assert lib.mcb_preference_loss(r, t, 16, 0.1, 0.0, 0, 16, 16, None, None, ws, None) == WORKSPACE
    assert lib.mcb_preference_loss(r, t, 16, 0.1, 0.0, 0, 16, 16, None, 16, 8, None) == WORKSPACE
    for beta, eps in ((0.0, 0.0), (math.nan, 0.0), (math.inf, 0.0), (0.1, -0.1), (0.1, 0.6), (0.1, math.nan)):
        assert lib.mcb_preference_loss(r, t, 16, beta, eps, 0, 16, 16, None, 16, ws, None) == SHAPE
        assert lib.mcb_preference_finish(16, t, 16, 16, 16, 16, 1, 3, 8, beta, eps, 0, None) == SHAPE
    assert lib.mcb_preference_loss(r, t, None, 0.1, 0.0, 0, 16, 16, None, 16, ws, None) == NULL
    assert lib.mcb_preference_finish(16, t, 16, 16, 16, 16, 1 << 31, 3, 8, 0.1, 0.0, 0, None) == SHAPE
    P = _lib.PolicyTerms
    for terms, code in ((P(None, 1, None, None, 0.2, 0.2, 0.0, 0), NULL), (P(16, 0, None, None, 0.2, 0.2, 0.0, 0), SHAPE),
                        (P(16, 1, None, None, -0.2, 0.2, 0.0, 0), SHAPE), (P(16, 1, None, None, 0.2, math.nan, 0.0, 0), SHAPE),
                        (P(16, 1, None, None, 0.2, 0.2, 0.1, 0), NULL), (P(16, 1, None, 16, 0.2, 0.2, -0.1, 0), SHAPE),
                        (P(16, 1, None, 16, 0.2, 0.2, math.inf, 0), SHAPE)):
        assert lib.mcb_policy_loss(r, t, C.byref(terms), 0, 16, 16, None, 16, ws, None) == code
        assert lib.mcb_policy_loss_rows(r, t, C.byref(terms), 16, 16, 16, None, None) == code
    T = _lib.TeacherTop
    for top, code in ((T(None, 16, 2, 8, 0), NULL), (T(16, None, 2, 8, 0), NULL), (T(16, 16, 0, 8, 0), SHAPE), (T(16, 16, 1025, 8, 0), SHAPE),
                      (T(16, 16, 2, 2, 0), UNSUPPORTED), (T(16, 16, 2, 8, 5), UNSUPPORTED)):
        assert lib.mcb_distill_loss(r, C.byref(top), None, 16, None, 16, ws, None) == code
        assert lib.mcb_distill_loss_rows(r, C.byref(top), 16, 16, None, None) == code
    assert lib.mcb_loss_weights(t, None, None, 2, 3, 8, 0, None) == NULL
    assert lib.mcb_loss_weights(t, None, 16, 0, 3, 8, 0, None) == SHAPE
    assert lib.mcb_loss_sums(16, 0, 1, 16, None) == SHAPE and lib.mcb_loss_sums(16, 4, 9, 16, None) == SHAPE
    assert lib.mcb_scale_rows(None, 16, 2, 2, 1, 0, None) == NULL and lib.mcb_scale_rows(16, 16, 2, 2, 0, 0, None) == SHAPE
    assert lib.mcb_token_loss_workspace_bytes(0, 3) == 0 and lib.mcb_token_loss_workspace_bytes(4, 100) >= 4 * 400 * 4
