"""Edges of the token scores and the distillation: what the header says of them, held to the letter."""
import numpy as np
import pytest
import torch

from tests.test_gpu_token_ops import TYPES, _check_distill_rows, _dev, _ids, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [40, 3000, 70001])
def test_teacher_entry_at_minus_inf_is_absent_whatever_its_id(kind, V):
    """The bounds are those of the same call with the absent entries named by an id of -1."""
    from image_caption_amd import ops
    rng = np.random.default_rng(V)
    N, K = 9, 70
    x = _logits(rng, N, V, kind)
    ti = rng.integers(0, V, (N, K))
    tl = (rng.standard_normal((N, K)) * 2).astype(np.float32)
    filler = [V, -100, 2 ** 31 - 1, -2 ** 31, V + 1]
    for n in range(5):                       # a padded list of 8, with each filler, and one past the first 64
        ti[n, 8:], tl[n, 8:] = filler[n], -np.inf
    ti[5, 69], tl[5, 69] = V, -np.inf
    ti[6], tl[6] = V, -np.inf                # no entries at all: loss 0 and a zero gradient
    ti[7, 3] = V                             # wrong, not absent
    ti[8, 3], tl[8, 3] = -5, np.nan
    g = rng.standard_normal(N).astype(np.float32)
    for t_kind in sorted(TYPES):
        t = _dev(tl, t_kind)
        loss, grad = ops.distill_loss(x, t, _ids(ti), 2.0, _dev(g))
        named = np.where(np.isneginf(tl), -1, ti)
        want_loss, want_grad = ops.distill_loss(x, t, _ids(named), 2.0, _dev(g))
        assert torch.equal(loss[:7], want_loss[:7]) and torch.equal(grad[:7], want_grad[:7])
        assert torch.isfinite(loss[:7]).all() and torch.isfinite(grad[:7].float()).all()
        assert loss[6] == 0 and not grad[6].any()
        assert loss[7:].isnan().all() and grad[7:].isnan().all()
        _check_distill_rows(x, t, named, 2.0, g, kind, ())
