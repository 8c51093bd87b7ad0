"""Refusals of the token operators that need no device: they come before any operand is looked at."""
import pytest
import torch


def _inputs(N=4, V=8):
    return torch.zeros(N, V), torch.zeros(N, dtype=torch.int32), torch.zeros(N, 2), torch.zeros(N)


def test_distillation_over_no_columns():
    from image_caption_amd import ops
    x, _, _, g = _inputs(4, 0)
    tl, ti = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    for grad in (None, g):
        with pytest.raises(ValueError, match="no columns"):
            ops.distill_loss(x, tl, ti, grad_loss=grad)
