"""Refusals of the token operators that need no device: they come before any operand is looked at."""
import pytest
import torch

WRAPS = 2 ** 32          # as a 32-bit integer: 0


def _inputs(N=4, V=8):
    return torch.zeros(N, V), torch.zeros(N, dtype=torch.int32), torch.zeros(N, 2), torch.zeros(N)


def test_distillation_over_no_columns():
    from image_caption_amd import ops
    x, _, _, g = _inputs(4, 0)
    tl, ti = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    for grad in (None, g):
        with pytest.raises(ValueError, match="no columns"):
            ops.distill_loss(x, tl, ti, grad_loss=grad)


def test_numbers_past_32_bits():
    """The library takes 32-bit sizes and ids; more must not come round to small ones."""
    from image_caption_amd import ops
    x, t, st, h = _inputs()
    for pad in (WRAPS, -WRAPS - 1, 2 ** 31):
        with pytest.raises(ValueError, match="pad_token"):
            ops.token_log_probs(x, t, pad_token=pad)
        with pytest.raises(ValueError, match="pad_token"):
            ops.token_log_probs_grad(x, t, st, h, h, pad_token=pad)
        with pytest.raises(ValueError, match="pad_token"):
            ops.embedding_scaled(x, t, pad_token=pad)
        with pytest.raises(ValueError, match="pad_token"):
            ops.embedding_grad(x, t, 10, pad_token=pad)
    with pytest.raises(ValueError, match="vocab_size"):
        ops.embedding_grad(x, t, WRAPS + 10)
    many = WRAPS + 4
    big, ids, st, h = (a[:1].expand(many, *a.shape[1:]) for a in (x, t, st, h))
    with pytest.raises(ValueError, match="rows"):
        ops.token_log_probs(big, ids)
    with pytest.raises(ValueError, match="rows"):
        ops.token_log_probs_grad(big, ids, st, h, out=big)
    with pytest.raises(ValueError, match="rows"):
        ops.distill_loss(big, st, st[:1].to(torch.int32).expand(many, 2))
    with pytest.raises(ValueError, match="rows"):
        ops.embedding_scaled(x, ids)
    with pytest.raises(ValueError, match="rows"):
        ops.embedding_grad(big, ids, 10)
