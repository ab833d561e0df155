"""LayerNormOp, the reference's operator."""
import pytest
import torch

from metal_candle_b200 import backend
from metal_candle_b200.backend import TrainingError
from tests.support import packed_reference as ref
from tests.test_gpu_packed_training import layer_norm_64, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_op(cuda_device, dtype):
    """No weight, no bias, the eps it was made with, the shape it is given."""
    x = rand(cuda_device, 3, 5, 33, seed=1, dtype=dtype)
    op = backend.LayerNormOp(0.25)
    assert op.name() == "layer-norm" and op.eps == 0.25
    y = op(x)
    assert y.shape == x.shape and y.dtype == dtype and torch.equal(y, backend.layer_norm_fused(x, eps=0.25))
    ref.check(y.view(15, 33), layer_norm_64(x, None, None, x, None, 0.25, dtype)["y"], "y")
    for bad in (x.cpu(), x.half(), x.transpose(0, 1), x[..., :0]):
        with pytest.raises(TrainingError):
            op(bad)
