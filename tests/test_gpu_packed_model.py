"""The model over packed documents: what it gives for each document by itself."""
import pytest
import torch

from metal_candle_b200.backend import TrainingError
from tests.test_gpu_post_training import REL, V, clones, close, small_model

pytestmark = pytest.mark.gpu

LENGTHS = [[9, 31, 20], [40, 17]]   # the second sequence ends in three tokens of padding
S = 60


def batch(dev, g):
    ids = torch.randint(0, V, (2, S), device=dev, generator=g)
    docs, targets = torch.full((2, S), -1, dtype=torch.int32, device=dev), torch.full((2, S), -1, device=dev)
    spans = []
    for b, lengths in enumerate(LENGTHS):
        at = 0
        for i, n in enumerate(lengths):
            docs[b, at:at + n] = i
            targets[b, at:at + n - 1] = ids[b, at + 1:at + n]
            spans.append((b, at, at + n))
            at += n
    return ids, docs, targets, spans


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_documents_by_themselves(cuda_device, dtype):
    model, _, _, g = small_model(cuda_device, dtype)
    ids, docs, targets, spans = batch(cuda_device, g)
    with model.packed(docs):
        logits = model.forward(ids)
        logp = model.token_log_probs(ids, targets)
        loss, grads = model.forward_backward(ids, targets)
        loss, grads = loss.clone(), clones(grads)
    total = int((targets >= 0).sum())
    want_loss, want = 0.0, [torch.zeros_like(t) for t in grads]
    for b, a, e in spans:
        alone = ids[b:b + 1, a:e].contiguous()
        close([logits[b, a:e]], [model.forward(alone)[0]], REL[dtype])
        close([logp[b, a:e]], [model.token_log_probs(alone, targets[b:b + 1, a:e].contiguous())[0]], REL[dtype])
        one, g1 = model.forward_backward(alone, targets[b:b + 1, a:e].contiguous())
        share = (e - a - 1) / total
        want_loss += float(one) * share
        want = [w + t * share for w, t in zip(want, g1)]
    assert abs(float(loss) - want_loss) <= REL[dtype] * want_loss
    close(grads, want, REL[dtype])
    # outside the block the sequence is one text again
    assert not torch.allclose(model.forward(ids)[0, 9:18], logits[0, 9:18], rtol=1e-2, atol=1e-2)


def test_a_prefix_is_read_in_both_directions(cuda_device):
    model, _, _, g = small_model(cuda_device, torch.float32)
    ids, docs, _, _ = batch(cuda_device, g)
    prefix = torch.zeros(2, S, dtype=torch.bool, device=cuda_device)
    prefix[0, 9:20] = True
    other = ids.clone()
    other[0, 19] = (other[0, 19] + 1) % V
    with model.packed(docs, prefix):
        a, b = model.forward(ids), model.forward(other)
    assert not torch.equal(a[0, 9], b[0, 9])                                        # sees the prefix's last token
    assert torch.equal(a[0, :9], b[0, :9]) and torch.equal(a[1], b[1])              # other documents do not
    with model.packed(docs):
        assert torch.equal(model.forward(ids)[0, 9:19], model.forward(other)[0, 9:19])


def test_refusals(cuda_device):
    model, ids, targets, _ = small_model(cuda_device, torch.bfloat16)
    docs = torch.zeros_like(ids)
    with model.packed(docs):
        with pytest.raises(TrainingError, match="positions"):
            model.forward(ids[:, :-1].contiguous())
        with pytest.raises(TrainingError, match="within packed"):
            model.capture_forward_backward(*ids.shape)
    with pytest.raises(TrainingError, match="document_ids is on cpu"):
        with model.packed(docs.cpu()):
            pass
    with pytest.raises(TrainingError, match="must be"):
        with model.packed(docs[0]):
            pass
    assert model._mask is None
    with pytest.raises(TrainingError, match="prefix"):
        with model.packed(docs, torch.zeros_like(docs[:, 1:], dtype=torch.uint8)):
            pass
    assert model._mask is None
    model.forward(ids[:, :-1].contiguous())


def test_blocks_within_blocks_and_after_an_error(cuda_device):
    model, ids, targets, _ = small_model(cuda_device, torch.bfloat16)
    one, many = torch.zeros_like(ids), torch.arange(ids.shape[1], device=cuda_device, dtype=ids.dtype).expand_as(ids).contiguous() // 4
    plain = model.forward(ids)
    with model.packed(many):
        apart = model.forward(ids)
        with model.packed(one):
            whole = model.forward(ids)
        assert torch.equal(model.forward(ids), apart)
    with pytest.raises(KeyError):
        with model.packed(many):
            raise KeyError("a step that failed")
    assert torch.equal(model.forward(ids), plain)
    assert not torch.equal(whole, apart) and torch.equal(whole[:, :4], apart[:, :4])
