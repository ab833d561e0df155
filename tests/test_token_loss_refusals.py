"""Refusals of the losses over given tokens that have tests of their own, on the CPU."""
import ctypes as C

from metal_candle_b200 import _lib
from tests.test_token_losses import ALIGN, rows, targets


def test_preference_workspace_alignment():
    """As mcb_policy_loss and mcb_distill_loss: on a 16-byte boundary."""
    lib = _lib.load()
    for at in (24, 20, 17):
        assert lib.mcb_preference_loss(C.byref(rows()), C.byref(targets()), 16, 0.1, 0.0, 0, 16, 16, None, at, 1 << 40, None) == ALIGN
