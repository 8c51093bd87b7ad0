"""Edges of the token scores and the distillation: what the header says of them, held to the letter."""
import numpy as np
import pytest
import torch

from tests.helpers import dev, np_of
from tests.test_gpu_token_ops import LOWEST, TYPES, _check_distill_rows, _dev, _f64, _ids, _logits

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


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [9, 3000])
@pytest.mark.parametrize("size", [1.0, 1e9, 1e20, 1e36])
def test_gradient_of_masked_columns_is_zero_however_large_the_entropy_weight(kind, V, size):
    """p log p is 0 where p is.  Elsewhere a weight past fp16's range may give infinities, never a NaN."""
    from image_caption_amd import ops
    rng = np.random.default_rng(V)
    N = 4
    x = rng.standard_normal((N, V)).astype(np.float32)
    masked = np.zeros((N, V), bool)
    masked[:, ::3] = True
    masked[3] = True
    masked[3, 1] = False                     # one column is left: its gradient is 0 as well
    x[masked] = -np.inf
    x[1, masked[1]] = LOWEST[kind]
    x = _dev(x, kind)
    tokens = _ids(np.ones(N))
    _, h, stats, _, _ = ops.token_log_probs(x, tokens)
    g_h = _dev(np.full(N, size))
    for g_lp in (None, _dev(np.ones(N))):
        for sign in (1, -1):
            got = ops.token_log_probs_grad(x, tokens, stats, h, g_lp, sign * g_h)
            assert not got[torch.as_tensor(masked, device=dev())].any()
            assert not got.isnan().any()


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [2, 3, 500, 3001, 30011, 140001])
@pytest.mark.parametrize("N", [5, 700])
def test_the_maximum_passes_a_nan_over(kind, V, N):
    """Rows of NaN beside -inf, beside the lowest value, beside numbers, and alone."""
    from image_caption_amd import ops
    if N * V > 1 << 24:
        N = 60
    rng = np.random.default_rng(V)
    x = rng.standard_normal((N, V)).astype(np.float32)
    x[0], x[1], x[2], x[3] = -np.inf, np.nan, LOWEST[kind], -np.inf
    x[0, V - 1] = x[2, 0] = x[4, V // 2] = np.nan
    want = np.where(np.isnan(x), -np.inf, _f64(_dev(x, kind))).max(1)
    x = _dev(x, kind)
    for top_k in (0, 2):
        lp, h, stats, ids, top = ops.token_log_probs(x, _ids(np.zeros(N)), top_k=top_k)
        np.testing.assert_array_equal(_f64(stats[:, 0]), want)
        nan = [0, 1, 2, 4]
        assert stats[nan, 1].isnan().all() and lp[nan].isnan().all() and h[nan].isnan().all()
        assert torch.equal(stats[3], stats.new_tensor([float("-inf"), 0])) and lp[3] == float("-inf") and h[3] == 0
        if top_k:
            np.testing.assert_array_equal(np_of(ids)[[0, 1, 3]], [[0, 1]] * 3)
            assert top[nan].isnan().all() and (top[3] == float("-inf")).all()
    ones = _dev(np.ones(N))
    got = ops.token_log_probs_grad(x, _ids(np.zeros(N)), stats, h, ones, ones)
    assert got[nan].isnan().all() and not got[3].any()
    assert torch.isfinite(got[5:].float()).all()
    loss, got = ops.distill_loss(x, _dev(np.zeros((N, 2))), _ids(np.zeros((N, 2))), 1.5, ones)
    assert loss[nan].isnan().all() and got[nan].isnan().all()
    assert loss[3] == float("inf") and not got[3].any()
    assert torch.isfinite(loss[5:]).all() and torch.isfinite(got[5:].float()).all()


@pytest.mark.parametrize("inside", [False, True])
def test_overwritten_logits_are_noticed_by_a_backward_pass(inside):
    """A graph that saved the logits must not go on with the gradient that took their place."""
    from image_caption_amd import ops
    N, V = 5, 60
    tokens, g = _ids(np.arange(N)), _dev(np.ones(N))
    for op in ("scores", "distillation"):
        w = torch.randn(N, V, device=dev(), requires_grad=True)
        x = w.exp()                              # whose backward pass reads x
        flat = x.detach()
        out = flat if inside else torch.empty_like(flat)
        if op == "scores":
            _, h, stats, _, _ = ops.token_log_probs(flat, tokens)
            ops.token_log_probs_grad(flat, tokens, stats, h, g, g, out=out)
        else:
            ops.distill_loss(flat, _dev(np.zeros((N, 2))), _ids(np.zeros((N, 2))), 1.0, g, out=out)
        if inside:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                x.sum().backward()
        else:
            x.sum().backward()
            assert torch.equal(w.grad, x.detach())


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_gradient_between_the_rows_of_the_logits(kind):
    """Logits and gradient side by side in the rows of one buffer."""
    from image_caption_amd import ops
    rng = np.random.default_rng(2)
    N, V, K = 7, 301, 5
    tokens, g = _ids(rng.integers(0, V, N)), _dev(rng.standard_normal(N))
    ti, tl = _ids(rng.integers(0, V, (N, K))), _logits(rng, N, K, "f32")
    for first, second in ((0, V), (V + 3, 2)):
        buf = _logits(rng, N, 2 * V + 3, kind)
        x, out = buf[:, first:first + V], buf[:, second:second + V]
        _, h, stats, _, _ = ops.token_log_probs(x, tokens)
        want = ops.token_log_probs_grad(x, tokens, stats, h, g, g)
        loss, d_want = ops.distill_loss(x, tl, ti, 2.0, g)
        keep = buf.clone()
        keep[:, second:second + V] = want
        assert ops.token_log_probs_grad(x, tokens, stats, h, g, g, out=out) is out and torch.equal(buf, keep)
        keep[:, second:second + V] = d_want
        again, d = ops.distill_loss(x, tl, ti, 2.0, g, out=out)
        assert d is out and torch.equal(again, loss) and torch.equal(buf, keep)
