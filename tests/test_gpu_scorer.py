"""SequenceScorer: scores of given sequences and their gradient, against the float64 restatement on the
policy's own logits, step by step."""
import numpy as np
import pytest
import torch

from tests import token_reference as ref
from tests.helpers import np_of, to_dev
from tests.test_gpu_searcher import _params, _searcher_modules, _sequences
from tests.token_reference import U

pytestmark = pytest.mark.gpu


def _step_logits(net, feats, seqs):
    """[B, T-1, V] float64: the policy called as a teacher-forced loop calls it."""
    state = net.reset_state(seqs, {"features": feats}, training=False)
    rows = []
    for t in range(1, seqs.shape[1]):
        pred, state = net((seqs[:, t - 1].contiguous(), {"features": feats}, state), training=False)
        rows.append(np_of(pred.reshape(seqs.shape[0], -1).double()))
    return np.stack(rows, 1)


@pytest.mark.parametrize("cell", ["lstm", "gru"])
@pytest.mark.parametrize("top_k", [0, 4])
def test_scores_of_given_sequences(cell, top_k):
    from image_caption_amd.utils.agent_utils import SequenceScorer
    dims = dict(F=24, D=8, E=8, H=32, V=40)
    net = _searcher_modules(_params(8, dims, cell, bias_seed=9), dims, cell)
    rng = np.random.default_rng(10)
    B, L, T = 6, 4, 9
    feats = to_dev(np.abs(rng.standard_normal((B, L, dims["D"]))).astype(np.float32))
    seqs = to_dev(_sequences(rng, B, T))
    scorer = SequenceScorer(net, pad_token=0, top_k=top_k)
    got = scorer((feats, seqs), training=False)
    x = _step_logits(net, feats, seqs)
    np.testing.assert_array_equal(np_of(got.logits.double()), x)
    tokens = np_of(seqs)[:, 1:]
    flat = x.reshape(-1, dims["V"])
    lp, h, _, ids, top = ref.score(flat, tokens.reshape(-1), 0, top_k)
    rel, D, log_s = ref.row_bounds(flat)
    bound = (rel + U * (6 * np.abs(log_s) + 3 * np.abs(flat).max(-1)) + 1e-30).reshape(B, T - 1)
    ref.check(np_of(got.log_probs), lp.reshape(B, T - 1), bound, "log_probs")
    ref.check(np_of(got.entropy), h.reshape(B, T - 1), bound * (2 + 3 * D.reshape(B, T - 1)), "entropy")
    if top_k:
        np.testing.assert_array_equal(np_of(got.top_ids), ids.reshape(B, T - 1, top_k))
    else:
        assert got.top_ids is None and got.top_log_probs is None
    a, b = rng.standard_normal((B, T - 1)).astype(np.float32), rng.standard_normal((B, T - 1)).astype(np.float32)
    g = scorer.grad(got, to_dev(a), to_dev(b))
    want = ref.score_grad(flat, tokens.reshape(-1), 0, a.reshape(-1).astype(np.float64), b.reshape(-1).astype(np.float64))
    # each gradient: a product of p (relative error of the sum and the exponent), two factors and a sum
    # of three terms below 2 + log V each
    size = (np.abs(a) + np.abs(b) * (2 + np.log(dims["V"])) * 2)[..., None]
    ref.check(np_of(g), want.reshape(x.shape), size * (2 * bound[..., None] + 16 * U), "gradient")
    only = scorer.grad(got, grad_entropy=to_dev(b))
    assert only.shape == g.shape and not torch.equal(only, g)


def test_scorer_refuses_sequences_of_one_token():
    from image_caption_amd.utils.agent_utils import SequenceScorer
    with pytest.raises(ValueError, match="after the first"):
        SequenceScorer(None)((torch.zeros(2, 3, 4), torch.zeros(2, 1, dtype=torch.int32)))
