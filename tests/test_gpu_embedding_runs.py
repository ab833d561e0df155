"""The token table's gradient where a token comes very often."""
import math

import pytest
import torch

from metal_candle_b200 import backend
from tests.support import packed_reference as ref
from tests.test_gpu_packed_training import embedding_64, rand

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
def test_a_token_that_comes_half_the_time(cuda_device, dtype):
    """Padding by an id at the end of a large vocabulary: the same sums, and no longer than by an id at its start, whose rows hold zeros already when
    the sums begin, or than as many different tokens."""
    M, H, V, hot = 65536, 896, 151936, 151645
    gen = torch.Generator(device=cuda_device).manual_seed(1)
    spread = torch.randint(0, V, (M,), device=cuda_device, generator=gen, dtype=torch.int32)
    ids = torch.where(torch.rand(M, device=cuda_device, generator=gen) < 0.5, torch.full_like(spread, hot), spread)
    ids[:300] = hot + 1 + torch.arange(300, device=cuda_device, dtype=torch.int32) % 3   # neighbours of it, a hundred times each
    dout = rand(cuda_device, M, H, seed=2, dtype=dtype)
    grad = backend.embedding_backward(ids, dout, V)
    part = torch.cat([torch.arange(24, device=cuda_device), torch.tensor([895], device=cuda_device)])
    ref.check(grad[:, part], embedding_64(ids, dout[:, part], V, 1.0), "grad")
    named = torch.zeros(V, dtype=torch.bool, device=cuda_device)
    named[ids.long()] = True
    assert not grad[~named].any()
    low = torch.where(ids == hot, torch.full_like(ids, 7), ids)
    even, start, late = (fastest(lambda: backend.embedding_backward(x, dout, V, grad=grad)) for x in (spread, low, ids))
    assert late <= 1.25 * start and max(start, late) <= 1.5 * even, (late, start, even)


def test_rows_named_once_and_often_side_by_side(cuda_device):
    """Every row of a stretch behind the first 64 MB of the table is named, by 1 to 400 tokens, up to the vocabulary's last; the rows
    between two named ones hold zeros."""
    H, V = 1024, 20000
    counts = [(1, 400, 2, 33, 32, 64, 0, 31, 96, 1, 0, 65)[r % 12] for r in range(700)]
    rows = torch.tensor([V - 700 + r for r, n in enumerate(counts) for _ in range(n)], device=cuda_device, dtype=torch.int64)
    ids = rows[torch.randperm(len(rows), device=cuda_device, generator=torch.Generator(device=cuda_device).manual_seed(1))]
    ids[::97] = -1
    dout = rand(cuda_device, len(ids), H, seed=3, dtype=BF16)
    grad = torch.full((V, H), math.nan, device=cuda_device)
    backend.embedding_backward(ids, dout, V, 0.5, grad=grad)
    ref.check(grad[:, :40], embedding_64(ids, dout[:, :40], V, 0.5), "grad")
    named = torch.zeros(V, dtype=torch.bool, device=cuda_device)
    named[ids[ids >= 0]] = True
    assert not grad[~named].any() and torch.isfinite(grad).all()


@pytest.mark.parametrize("dtype,H", [(BF16, 896), (F32, 896), (F32, 130), (BF16, 64), (F32, 17), (BF16, 2056)])
def test_runs_of_any_length_from_any_place(cuda_device, dtype, H):
    """Runs of a few to a thousand parts (8 tokens each), ending and beginning at the parts' borders and between, one behind the other; alone in
    the batch; with gradients added to."""
    parts = [1, 2, 7, 8, 9, 15, 16, 17, 62, 63, 64, 65, 66, 127]
    lengths = [8 * n + off for n in parts for off in (0, 1, 7)] + [3, 5]
    order = torch.randperm(len(lengths), generator=torch.Generator().manual_seed(H)).tolist()
    V = len(lengths) + 3
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    for sizes in ([lengths[i] for i in order], [8 * 512], [8 * 513 + 1, 8 * 300], [513, 8 * 64 + 1, 519]):
        ids = torch.cat([torch.full((n,), i + 1, device=cuda_device, dtype=torch.int32) for i, n in enumerate(sizes)])
        assert len(ids) <= 16384
        ids = ids[torch.randperm(len(ids), device=cuda_device, generator=gen)]
        dout = rand(cuda_device, len(ids), H, seed=4, dtype=dtype)
        value = embedding_64(ids, dout, V, 3.0)
        grad = backend.embedding_backward(ids, dout, V, 3.0)
        ref.check(grad, value, "grad")
        assert torch.equal(grad, backend.embedding_backward(ids, dout, V, 3.0))
        before = rand(cuda_device, V, H, seed=5)
        more = backend.embedding_backward(ids, dout, V, 3.0, grad=before.clone(), accumulate=True)
        at = before.cpu().double()
        ref.check(more, (at + value[0], value[1] + 2.0 ** -24 * (at.abs() + value[0].abs())), "accumulated")


def test_one_token_alone(cuda_device):
    """All of 300000 tokens the same: parts of 32, some ten thousand of them."""
    M, H = 300000, 96
    ids = torch.full((M,), 2, device=cuda_device, dtype=torch.int32)
    dout = rand(cuda_device, M, H, seed=6, dtype=BF16)
    ref.check(backend.embedding_backward(ids, dout, 4), embedding_64(ids, dout, 4, 1.0), "grad")
