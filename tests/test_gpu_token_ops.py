"""Token scores, distillation and the scaled embedding with their gradients against the float64
restatement of tests/token_reference.py, with bounds that count roundings."""
import numpy as np
import pytest
import torch

from tests import token_reference as ref
from tests.helpers import dev, np_of
from tests.token_reference import HALF_STEP, TINY, U

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOWEST = {k: float(torch.finfo(t).min) for k, t in TYPES.items()}


def _dev(x, kind="f32"):
    return torch.as_tensor(np.asarray(x), device=dev()).to(TYPES[kind])


def _ids(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32, device=dev())


def _f64(t):
    return np_of(t.double())


def _logits(rng, N, V, kind, spread=3.0):
    return _dev((rng.standard_normal((N, V)) * spread).astype(np.float32), kind)


def _check_score(x, tokens, pad=-1, k=0, what="", top_k_out=None):
    """Runs the operator on x and holds every output to the reference; returns the outputs."""
    from image_caption_amd import ops
    got = ops.token_log_probs(x, _ids(tokens), top_k=k, pad_token=pad)
    X, t = _f64(x).reshape(-1, x.shape[-1]), np.asarray(tokens).reshape(-1)
    lp, h, stats, ids, top = ref.score(X, t, pad, k)
    rel, D, log_s = ref.row_bounds(X)
    m = np.where(np.isfinite(stats[:, 0]), stats[:, 0], 0.0)
    with np.errstate(all="ignore"):
        flat = lambda v, n=None: np_of(v).reshape(len(t), *((n,) if n is not None else ()))    # noqa: E731
        d_t = np.abs(X[np.arange(len(t)), np.clip(t, 0, X.shape[1] - 1)] - m)
        base = rel + 4 * U * np.abs(log_s)
        ref.check(flat(got[0]), lp, base + U * (d_t + 2 * np.abs(lp)), what + " log_probs")
        ref.check(flat(got[1]), h, rel * (1 + 2 * D) + 4 * U * (np.abs(log_s) + D), what + " entropy")
        ref.check(flat(got[2], 2)[:, 0], stats[:, 0], 0.0, what + " maximum")
        ref.check(flat(got[2], 2)[:, 1], stats[:, 1], base, what + " log of the sum")
        if k:
            np.testing.assert_array_equal(flat(got[3], k), ids, err_msg=what + " alternatives")
            ref.check(flat(got[4], k), top, base[:, None] + 4 * U * (np.abs(top) + np.abs(log_s)[:, None]),
                      what + " alternatives' log probabilities")
    return got


def _grad_bound(X, g_lp, g_h, kind, g):
    lp, p, m, log_s, none = ref.softmax_rows(X)
    rel, D, _ = ref.row_bounds(X)
    with np.errstate(all="ignore"):
        d = np.abs(X - m[:, None])
        rel_p = (rel + 6 * U * np.abs(log_s))[:, None] + U * (4.5 * d + 4)
        h = -np.where(p > 0, p * lp, 0.0).sum(-1)[:, None]
        u = np.where(p > 0, lp + h, 0.0)
        err_u = U * (d + 6 * np.abs(log_s)[:, None] + 4 * h) + (rel * (2 + 2 * D))[:, None]
        a, b = np.abs(g_lp)[:, None], np.abs(g_h)[:, None]
        noise = np.where(p > 0, p * ((a + b * np.abs(u)) * (rel_p + 4 * U) + b * err_u), 0.0)
        return noise + 2 * U * a + HALF_STEP[kind] * np.abs(g) * (1 + 1e-3) + TINY[kind] + 1e-37


def _check_score_grad(x, tokens, stats, entropy, g_lp, g_h, pad=-1, kind="f32", what="", out=None):
    from image_caption_amd import ops
    X, t = _f64(x).reshape(-1, x.shape[-1]), np.asarray(tokens).reshape(-1)
    shape = x.shape[:-1]
    got = ops.token_log_probs_grad(x, _ids(tokens), stats, entropy,
                                   None if g_lp is None else _dev(g_lp).reshape(shape),
                                   None if g_h is None else _dev(g_h).reshape(shape), pad_token=pad, out=out)
    zero = np.zeros(len(t))
    a, b = (zero if g is None else np.asarray(g, np.float32).astype(np.float64).reshape(-1) for g in (g_lp, g_h))
    want = ref.score_grad(X, t, pad, a, b)
    assert got.dtype == x.dtype and got.shape == x.shape
    ref.check(_f64(got).reshape(X.shape), want, _grad_bound(X, a, b, kind, want), what + " gradient")
    return got


SIZES = [1, 2, 3, 4, 5, 7, 8, 9, 31, 63, 64, 65, 255, 256, 257, 511, 1000, 1023, 1025, 2048, 4099, 5000, 10000, 16385]


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", SIZES)
def test_scores_and_gradient(kind, V):
    rng = np.random.default_rng(V)
    for N in (1, 2, 7):
        x = _logits(rng, N, V, kind)
        tokens = rng.integers(0, V, N)
        out = _check_score(x, tokens, k=min(V, 32), what="N=%d V=%d" % (N, V))
        g_lp, g_h = rng.standard_normal(N), rng.standard_normal(N)
        _check_score_grad(x, tokens, out[2], out[1], g_lp, g_h, kind=kind, what="N=%d V=%d" % (N, V))
        _check_score_grad(x, tokens, out[2], out[1], g_lp, None, kind=kind)
        _check_score_grad(x, tokens, out[2], out[1], None, g_h, kind=kind)


@pytest.mark.parametrize("kind,V", [("f32", 32768), ("f32", 50000), ("bf16", 50001), ("f16", 65535), ("f32", 65537),
                                    ("f32", 131071), ("bf16", 131073), ("f16", 262145)])
@pytest.mark.parametrize("N", [1, 3, 40])
def test_scores_and_gradient_of_large_vocabularies(kind, V, N):
    rng = np.random.default_rng(V + N)
    x = _logits(rng, N, V, kind)
    tokens = rng.integers(0, V, N)
    tokens[0] = V - 1
    out = _check_score(x, tokens, k=16)
    g_lp, g_h = rng.standard_normal(N), rng.standard_normal(N)
    _check_score_grad(x, tokens, out[2], out[1], g_lp, g_h, kind=kind)


@pytest.mark.parametrize("kind,N,V", [("f32", 1400, 3000), ("bf16", 800, 5000), ("f16", 2699, 3000), ("f32", 300, 1000), ("bf16", 2100, 257), ("f16", 600, 2000), ("f32", 5000, 33)])
def test_scores_of_many_rows(kind, N, V):
    rng = np.random.default_rng(N)
    x = _logits(rng, N, V, kind)
    tokens = rng.integers(0, V, N)
    tokens[rng.random(N) < 0.3] = 0
    out = _check_score(x, tokens, pad=0, k=5)
    _check_score_grad(x, tokens, out[2], out[1], rng.standard_normal(N), rng.standard_normal(N), pad=0, kind=kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [5, 300, 5000, 70001])
def test_masked_logits(kind, V):
    """-inf and the type's lowest value among the logits, rows of nothing else, NaN and +inf, rows of
    the padding token that hold NaN, tokens outside the vocabulary."""
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((17, V)) * 2).astype(np.float32)
    x[0, rng.random(V) < 0.5] = -np.inf
    x[0, V // 2] = 1.0
    x[1, rng.random(V) < 0.5] = LOWEST[kind]
    x[2] = -np.inf                                # nothing left
    x[3] = LOWEST[kind]                           # all alike
    x[4] = -np.inf
    x[4, V - 1] = 3.0                             # one left
    x[5, V // 3] = np.nan
    x[6, V // 3] = np.inf
    x[7] = np.nan                                 # behind the padding token
    x[8], x[9] = 0.0, -0.0
    x[9, ::2] = 0.0
    x[10, 0] = LOWEST[kind]
    x[11] = -np.inf
    x[12] = LOWEST[kind]
    x[12, 1] = -np.inf
    x[13] *= 30 if kind == "f16" else 1e4
    x[14] *= 1 if kind == "f16" else 1e9          # rate * x rounds off what tells the elements apart
    x[15] *= 1 if kind == "f16" else 1e30
    x[16] -= 1 if kind == "f16" else 1e8
    tokens = np.array([V // 2, 1, 0, 2, V - 1, 1, 1, 0, 3, 4, 0, V, 1, 2, 1, 2, 3])
    tokens[2] = 1
    tokens[10] = 4
    pad = 0
    xd = _dev(x, kind)
    out = _check_score(xd, tokens, pad=pad, k=min(V, 9))
    g = np.full(17, 0.5)
    _check_score_grad(xd, tokens, out[2], out[1], g, -g, pad=pad, kind=kind)
    for bad in (-1, -7, V, V + 5, 2 ** 31 - 1, -2 ** 31):
        t = np.full(17, bad)
        t[7] = pad
        out = _check_score(xd, t, pad=pad, k=1)
        _check_score_grad(xd, t, out[2], out[1], g, None, pad=pad, kind=kind)
        _check_score_grad(xd, t, out[2], out[1], None, g, pad=pad, kind=kind)
    zero = np.zeros(17)
    zero[0] = 1.0                                 # gradients of zero leave rows of NaN at zero
    _check_score_grad(xd, tokens, out[2], out[1], zero, zero * 0, pad=pad, kind=kind)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [40, 1024, 10000, 50001, 140000])
def test_alternatives_among_ties_and_in_any_order(kind, V):
    """Equal logits go to the lower id; the best ones may lie anywhere, also all in the columns that
    one lane reads."""
    rng = np.random.default_rng(V)
    ramp = np.linspace(-4, 4, V).astype(np.float32)
    rows = [np.zeros(V), np.full(V, LOWEST[kind]), ramp, ramp[::-1], rng.integers(0, 3, V) * 1.0,
            np.where(np.arange(V) == V - 1, 1.0, 0.0), np.where(np.arange(V) == 0, -1.0, 0.0)]
    for stride in (4, 8, 256, 512, 1024, 2048, 4096, 8192):
        r = rng.standard_normal(V) * 0.1
        r[3::stride] += 5.0 + rng.integers(0, 2, len(r[3::stride]))
        rows.append(r)
    for width in (8, 64, 300):
        r = rng.standard_normal(V) * 0.1
        r[V // 3:V // 3 + width] += 5.0
        rows.append(r)
    few = np.full(V, -np.inf)
    few[rng.permutation(V)[:5]] = 1.0
    rows.append(few)
    x = _dev(np.stack(rows).astype(np.float32), kind)
    for k in (1, 2, 31, 32):
        _check_score(x, rng.integers(0, V, len(rows)), k=k)


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [7, 100, 2049, 40003, 270001])
def test_alternatives_of_rows_with_few_columns_left(kind, V):
    """Vocabularies masked but for some columns, to -inf, to the type's lowest value or to NaN: the
    columns left over follow those in order, also where whole shares of a row have none."""
    rng = np.random.default_rng(V + 1)
    rows = []
    for left in (0, 1, 5, 31, 32, 40, 129, 700, 5000):
        for gone in (-np.inf, LOWEST[kind]):
            for level in (0.0, 1.0):              # the same value everywhere, or spread
                r = np.full(V, gone)
                at = rng.permutation(V)[:left]
                r[at] = 2.0 + level * rng.standard_normal(len(at))
                rows.append(r)
    for lo, hi in ((0, V // 9), (V // 2, V), (V - 3, V), (V // 3, V // 3 + 2)):
        r = np.full(V, -np.inf)
        r[lo:hi] = rng.standard_normal(hi - lo)
        rows.append(r)
        rows.append(np.where(np.isinf(r), LOWEST[kind], r))
    r = np.full(V, -np.inf)                       # lowest values and -inf, nothing else
    r[::3] = LOWEST[kind]
    rows.append(r)
    r = rng.standard_normal(V)                    # the better half stands behind, its values alike
    r[V // 2:] = 9.0
    rows.append(r)
    r = np.where(rng.random(V) < 0.5, 0.0, -0.0)
    rows.append(r)
    x = np.stack(rows).astype(np.float32)
    tokens = rng.integers(0, V, len(rows))
    for k in (1, min(V, 6), min(V, 32)):
        _check_score(_dev(x, kind), tokens, k=k, what="V=%d k=%d" % (V, k))
        _check_score(_dev(x[-1:], kind), tokens[-1:], k=k)
    _check_score(_dev(np.concatenate([x] * 20)[:, :min(V, 2049)], kind), np.tile(tokens % min(V, 2049), 20), k=min(V, 7))


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [3, 500, 30011])
def test_rows_of_nan(kind, V):
    """Rows of NaN alone, or of NaN and -inf: no number comes out of them, and nothing but them."""
    from image_caption_amd import ops
    rng = np.random.default_rng(V)
    x = rng.standard_normal((4, V)).astype(np.float32)
    x[1] = np.nan
    x[2] = -np.inf
    x[2, V // 2] = np.nan
    tokens, k = rng.integers(0, V, 4), min(V, 6)
    xd = _dev(x, kind)
    lp, h, stats, ids, top = ops.token_log_probs(xd, _ids(tokens), top_k=k)
    g = ops.token_log_probs_grad(xd, _ids(tokens), stats, h, torch.ones_like(lp), torch.ones_like(h))
    loss, dg = ops.distill_loss(xd, torch.zeros(4, 2, device=dev()), _ids(rng.integers(0, V, (4, 2))), 1.5,
                                torch.ones_like(lp))
    for got in (lp, h, stats[:, 1], top, g, loss, dg):
        nan = torch.isnan(got).reshape(4, -1)
        assert nan[1:3].all() and not nan[[0, 3]].any()
    np.testing.assert_array_equal(np_of(ids)[1:3], [list(range(k))] * 2)


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_rows_apart_from_each_other(kind):
    """Leading dimensions, the first positions of a [B,T,V] tensor, transposed and broadcast rows."""
    rng = np.random.default_rng(5)
    V = 301
    buf = _logits(rng, 12, 333, kind)
    cube = _logits(rng, 24, V, kind).view(4, 6, V)
    line = _logits(rng, 1, V, kind)
    for x in (buf[:, :V], buf[:, 32:], buf[::2, 1:V + 1], cube[:, :-1], cube[:, 1:4], cube.transpose(0, 1),
              cube[::2, ::3], line.expand(5, V), line.view(V), cube[:, :, 1:300], cube[1:2, 2:5]):
        shape = x.shape[:-1]
        tokens = rng.integers(0, x.shape[-1], shape)
        out = _check_score(x, tokens, k=4, what=str(tuple(x.stride())))
        g_lp, g_h = rng.standard_normal(shape), rng.standard_normal(shape)
        _check_score_grad(x, tokens, out[2], out[1], g_lp, g_h, kind=kind, what=str(tuple(x.stride())))
    with pytest.raises(ValueError, match="contiguous rows"):
        from image_caption_amd import ops
        ops.token_log_probs(buf[:, ::2], _ids(np.zeros(12)))


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [129, 9000, 70003])
def test_gradients_in_place_and_into_views(kind, V):
    rng = np.random.default_rng(V)
    from image_caption_amd import ops
    N = 6
    buf = _logits(rng, N, V + 13, kind)
    x = buf[:, 5:V + 5]
    tokens = rng.integers(0, V, N)
    keep = buf.clone()
    out = ops.token_log_probs(x, _ids(tokens))
    g_lp, g_h = _dev(rng.standard_normal(N)), _dev(rng.standard_normal(N))
    apart = ops.token_log_probs_grad(x, _ids(tokens), out[2], out[1], g_lp, g_h)
    tl, ti = _logits(rng, N, 7, kind), _ids(rng.integers(0, V, (N, 7)))
    loss, d_apart = ops.distill_loss(x, tl, ti, 2.0, g_lp)
    view = torch.zeros(N, V + 40, dtype=x.dtype, device=dev())
    ops.token_log_probs_grad(x, _ids(tokens), out[2], out[1], g_lp, g_h, out=view[:, 3:V + 3])
    assert torch.equal(view[:, 3:V + 3], apart) and not view[:, :3].any() and not view[:, V + 3:].any()
    same = ops.token_log_probs_grad(x, _ids(tokens), out[2], out[1], g_lp, g_h, out=x)
    assert same is x and torch.equal(x, apart)
    assert torch.equal(buf[:, :5], keep[:, :5]) and torch.equal(buf[:, V + 5:], keep[:, V + 5:])
    buf.copy_(keep)
    loss2, d2 = ops.distill_loss(x, tl, ti, 2.0, g_lp, out=x)
    assert torch.equal(loss, loss2) and torch.equal(d2, d_apart)
    assert torch.equal(buf[:, :5], keep[:, :5]) and torch.equal(buf[:, V + 5:], keep[:, V + 5:])


@pytest.mark.parametrize("N,V", [(600, 1001), (600, 9000), (40, 9000), (7, 70001), (40, 50000)])
def test_the_same_call_gives_the_same_bits(N, V):
    """Every thread of a workgroup that writes a result has to hold the same statistics."""
    from image_caption_amd import ops
    rng = np.random.default_rng(N)
    x, tokens = _logits(rng, N, V, "bf16"), _ids(rng.integers(0, V, N))
    ti, tl, g = _ids(rng.integers(0, V, (N, 70))), _logits(rng, N, 70, "f32"), _dev(rng.standard_normal(N))
    first = ops.token_log_probs(x, tokens, top_k=32) + ops.distill_loss(x, tl, ti, 2.0, g)
    for _ in range(8):
        again = ops.token_log_probs(x, tokens, top_k=32) + ops.distill_loss(x, tl, ti, 2.0, g)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_offsets_past_32_bits():
    """Rows that start 2^31 elements and more behind the first."""
    from image_caption_amd import ops
    rng = np.random.default_rng(3)
    ld, V = (1 << 30) + 8, 1001
    buf = torch.zeros(2 * ld + 8192, dtype=torch.bfloat16, device=dev())
    x = buf.as_strided((3, V), (ld, 1))
    rows = _logits(rng, 3, V, "bf16")
    x.copy_(rows)
    tokens = rng.integers(0, V, 3)
    a = ops.token_log_probs(x, _ids(tokens), top_k=3)
    b = ops.token_log_probs(rows, _ids(tokens), top_k=3)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = _dev(np.ones(3))
    want = ops.token_log_probs_grad(rows, _ids(tokens), b[2], b[1], g, g)
    ops.token_log_probs_grad(x, _ids(tokens), b[2], b[1], g, g, out=x)
    assert torch.equal(x, want)
    table = buf[:524289 * 4096].view(524289, 4096)               # the last row starts at 2^31
    table[-1] = 3.0
    table[0] = 2.0
    got = ops.embedding_scaled(table, _ids([524288, 0, 524289]), scale=0.5)
    assert (got[0] == 1.5).all() and (got[1] == 1.0).all() and not got[2].any()


# ---- distillation --------------------------------------------------------------------------

def _check_distill(x, tl, ti, tau, g=None, kind="f32", what=""):
    from image_caption_amd import ops
    loss, grad = ops.distill_loss(x, tl, _ids(ti), temperature=tau, grad_loss=None if g is None else _dev(g).reshape(x.shape[:-1]))
    X, T, I = _f64(x).reshape(-1, x.shape[-1]), _f64(tl).reshape(-1, tl.shape[-1]), np.asarray(ti).reshape(-1, tl.shape[-1])
    tau = float(np.float32(tau))
    G = None if g is None else np.asarray(g, np.float32).astype(np.float64).reshape(-1)
    want, want_g = ref.distill(X, T, I, tau, G)
    rel, D, log_s = ref.row_bounds(X, tau)
    lp, p, m, _, none = ref.softmax_rows(X, tau)
    N, K = I.shape
    bound, q_sum = np.zeros(N), np.zeros_like(X)
    rel_q = np.zeros(N)
    with np.errstate(all="ignore"):
        for n in range(N):
            there = (I[n] >= 0) & (I[n] < X.shape[1]) & np.isfinite(T[n])
            if not there.any():
                continue
            t = T[n][there] / tau
            spread = np.abs(t - t.max())
            q = np.exp(t - t.max())
            q /= q.sum()
            log_q = np.log(np.maximum(q, 1e-300))
            rel_q[n] = U * (K / 64 + 12 + 4.5 * (q * spread).sum() + 4) 
            l = lp[n, I[n][there]]
            d = np.abs(X[n, I[n][there]] - m[n]) / tau
            err = U * (3 * spread + 4 * np.log(K + 1) + 2 * np.abs(log_q)) + rel_q[n]          # of log q
            err = err + U * (3 * d + 4 * abs(log_s[n]) + 2 * np.abs(l)) + rel[n]                # and of log p
            size = np.where(q > 0, np.abs(log_q - l), 0.0)
            each = rel_q[n] + U * (4.5 * spread + K / 64 + 16)
            bound[n] = tau * tau * (np.where(q > 0, q * (err + size * each), 0.0)).sum() + 4 * U * abs(want[n])
            np.add.at(q_sum[n], I[n][there], q)
        ref.check(np_of(loss).reshape(-1), want, np.where(np.isfinite(bound), bound, 0.0), what + " loss")
        if g is None:
            assert grad is None
            return
        d = np.abs(X - m[:, None]) / tau
        rel_p = (rel + 4 * U)[:, None] + 4.5 * U * np.where(p > 0, d, 0.0)
        b = np.abs(G)[:, None] * tau * (p * rel_p + q_sum * (rel_q[:, None] + U * (4.5 * 60 + K)) + 4 * U * (p + q_sum))
    b = np.where(np.isfinite(b), b, 0.0) + HALF_STEP[kind] * np.abs(np.where(np.isfinite(want_g), want_g, 0)) * (1 + 1e-3)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    ref.check(_f64(grad).reshape(X.shape), want_g, b + TINY[kind] + 1e-37, what + " gradient")


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [1, 3, 8, 65, 257, 1000, 5000, 10000, 16387, 50001, 66000, 131079])
def test_distillation(kind, V):
    rng = np.random.default_rng(V)
    for N, K, tau in ((1, 1, 1.0), (3, 8, 2.0), (5, 20, 0.5), (2, 256, 3.7), (9, 65, 1.0)):
        K = min(K, V)
        x = _logits(rng, N, V, kind)
        ti = np.stack([rng.permutation(V)[:K] for _ in range(N)])
        tl = _logits(rng, N, K, ["f32", "bf16", "f16"][K % 3])
        g = rng.standard_normal(N)
        _check_distill(x, tl, ti, tau, g, kind, "N=%d K=%d" % (N, K))
        _check_distill(x, tl, ti, tau, None, kind, "N=%d K=%d" % (N, K))


@pytest.mark.parametrize("kind,V", [("f32", 5), ("f32", 1000), ("f32", 2047), ("f32", 4001), ("f32", 9000), ("f32", 10243),
                                    ("f32", 28675), ("f32", 30000), ("bf16", 2049), ("bf16", 4095), ("bf16", 8191),
                                    ("f16", 20481), ("bf16", 53247), ("f16", 53255), ("bf16", 60000)])
def test_distillation_of_many_rows(kind, V):
    """Every division of a row over waves and registers that a batch of over 512 rows takes."""
    rng = np.random.default_rng(V)
    N, K = 520, min(V, 20)
    x = _logits(rng, N, V, kind)
    x[::7, ::3] = float("-inf")
    ti = rng.integers(0, V, (N, K))
    ti[::7] = ti[::7] // 3 * 3 + 1 if V > 5 else 1
    ti = np.minimum(ti, V - 1)
    ti[rng.random(N) < 0.2] = -1
    _check_distill(x, _logits(rng, N, K, "f32"), ti, 2.0, rng.standard_normal(N), kind)


@pytest.mark.parametrize("in_place", [False, True])
def test_streams_past_the_caches_give_the_same_bits(in_place):
    """Calls so large that they go past the caches, against the same rows in smaller calls."""
    from image_caption_amd import ops
    g = torch.Generator(device=dev())
    g.manual_seed(1)
    x = torch.randn(5500, 20000, device=dev(), generator=g)
    tokens = torch.randint(0, 20000, (5500,), device=dev(), generator=g, dtype=torch.int32)
    for k in (0, 5):
        whole = ops.token_log_probs(x, tokens, top_k=k)
        for r in (slice(0, 2750), slice(2750, 5500)):
            part = ops.token_log_probs(x[r], tokens[r], top_k=k)
            assert all(torch.equal(a[r], b) for a, b in zip(whole, part) if b is not None)
    lp, h, stats = whole[:3]
    a, b = (torch.randn(5500, device=dev(), generator=g) for _ in range(2))
    ti = torch.randint(-1, 20000, (5500, 30), device=dev(), generator=g, dtype=torch.int32)
    tl = torch.randn(5500, 30, device=dev(), generator=g)
    parts = [slice(i, i + 1100) for i in range(0, 5500, 1100)]
    small = torch.cat([ops.token_log_probs_grad(x[r], tokens[r], stats[r], h[r], a[r], b[r]) for r in parts])
    y = x.clone() if in_place else x
    assert torch.equal(ops.token_log_probs_grad(y, tokens, stats, h, a, b, out=y if in_place else None), small)
    pairs = [ops.distill_loss(x[r], tl[r], ti[r], 1.5, a[r]) for r in parts]
    y = x.clone() if in_place else x
    loss, grad = ops.distill_loss(y, tl, ti, 1.5, a, out=y if in_place else None)
    assert torch.equal(loss, torch.cat([p[0] for p in pairs])) and torch.equal(grad, torch.cat([p[1] for p in pairs]))
    del x, y, small, grad, pairs
    table = torch.randn(3000, 256, device=dev(), generator=g)
    ids = torch.randint(-2, 3002, (120000,), device=dev(), generator=g, dtype=torch.int32)
    rows = ops.embedding_scaled(table, ids, scale=3.0, pad_token=7)
    assert torch.equal(rows, torch.cat([ops.embedding_scaled(table, i, scale=3.0, pad_token=7) for i in ids.split(60000)]))
    got = ops.embedding_grad(rows, ids, 3000, scale=0.5, pad_token=7)
    keep = (ids >= 0) & (ids < 3000) & (ids != 7)
    want = torch.zeros(3000, 256, device=dev(), dtype=torch.float64)
    want.index_add_(0, ids[keep].long(), rows[keep].double())
    size = torch.zeros_like(want).index_add_(0, ids[keep].long(), rows[keep].double().abs())
    count = torch.bincount(ids[keep].long(), minlength=3000).double()[:, None]
    assert ((got.double() - 0.5 * want).abs() <= U * (count + 2) * size).all()


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("V", [50, 3000, 70001])
def test_distillation_entries_that_are_absent_double_or_wrong(kind, V):
    rng = np.random.default_rng(V)
    K, N = 6, 20
    x = (rng.standard_normal((N, V)) * 2).astype(np.float32)
    ti = np.stack([rng.permutation(V)[:K] for _ in range(N)])
    tl = (rng.standard_normal((N, K)) * 2).astype(np.float32)
    ti[0] = -1                                    # no entries
    ti[1, 2:] = -1
    tl[1, 3] = np.nan                             # NaN in an absent entry
    tl[2] = -np.inf                               # no entries either
    tl[3, 1:4] = -np.inf
    ti[4] = 7                                     # the same id in every entry
    ti[5, 3:] = ti[5, :3]                         # doubled
    ti[6, 2] = V                                  # outside
    ti[7, 0] = -2
    x[8] = -np.inf                                # the student has no distribution
    x[9] = np.nan
    x[10, 4] = np.inf
    x[11, ti[11, 2]] = -np.inf                    # the teacher wants what the student has masked
    x[12, :V // 2] = LOWEST[kind]
    ti[12] = V // 2 + np.arange(K)
    tl[13, 2] = np.nan
    x[14] = np.nan                                # behind a row without entries
    ti[14] = -1
    tl[15] = LOWEST["f16"]
    x[16] = LOWEST[kind]
    if kind != "f16":
        x[17] *= 1e9
        x[18] *= 1e30
        x[19] -= 1e8
    for g in (np.ones(N), np.where(np.arange(N) % 2, 0.0, -1.5), None):
        want_nan = g is not None
        _check_distill_rows(_dev(x, kind), _dev(tl), ti, 2.0, g, kind, skip_grad=[13] if want_nan else [])


def _check_distill_rows(x, tl, ti, tau, g, kind, skip_grad):
    """Row by row, so that a row whose NaN only the loss defines (a NaN among the teacher's logits makes
    the gradient NaN at the teacher's ids alone) is checked by hand."""
    from image_caption_amd import ops
    for n in range(x.shape[0]):
        gn = None if g is None else g[n:n + 1]
        if n in skip_grad:
            loss, grad = ops.distill_loss(x[n:n + 1], tl[n:n + 1], _ids(ti[n:n + 1]), tau, _dev(gn))
            assert np.isnan(np_of(loss)).all()
            assert bool(torch.isnan(grad).any()) == bool(gn[0] != 0)
            continue
        _check_distill(x[n:n + 1], tl[n:n + 1], ti[n:n + 1], tau, gn, kind, "row %d" % n)


def test_distillation_of_views_and_extreme_temperatures():
    rng = np.random.default_rng(11)
    cube = _logits(rng, 20, 77, "f32").view(4, 5, 77)
    tl, ti = _logits(rng, 16, 3, "f32").view(4, 4, 3), rng.integers(0, 77, (4, 4, 3))
    for tau in (0.001, 0.1, 1000.0):
        _check_distill(cube[:, :-1], tl, ti, tau, rng.standard_normal((4, 4)))
    _check_distill(cube[0, 0], tl[0, 0], ti[0, 0], 1.0, np.ones(()))


# ---- embedding -----------------------------------------------------------------------------

@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("D", [1, 3, 8, 63, 64, 100, 256, 257, 512, 513, 1500, 2048])
def test_scaled_lookup(kind, D):
    from image_caption_amd import ops
    rng = np.random.default_rng(D)
    V = 50
    table = _logits(rng, V, D, kind)
    for shape in ((1,), (7,), (3, 9), (0,), (2, 0), ()):
        ids = rng.integers(-2, V + 2, shape)
        got = ops.embedding_scaled(table, _ids(ids), scale=22.627417, pad_token=4)
        assert tuple(got.shape) == (*shape, D) and got.dtype == table.dtype
        want = _f64(table)[np.clip(ids, 0, V - 1)] * float(np.float32(22.627417))
        want[(ids < 0) | (ids >= V) | (ids == 4)] = 0.0
        # one product in float32 and one rounding to the type
        ref.check(_f64(got), want, np.abs(want) * (U + HALF_STEP[kind]) * (1 + 1e-3) + TINY[kind])
    table[3] = float("nan")                       # NaN of a row that is padding stays behind
    assert not ops.embedding_scaled(table, _ids([3, 3]), pad_token=3).any()


def _check_embed_grad(grad, ids, V, scale, pad, kind, what=""):
    from image_caption_amd import ops
    D = grad.shape[-1]
    got = ops.embedding_grad(grad, _ids(ids), V, scale=scale, pad_token=pad)
    G, I = _f64(grad).reshape(-1, D), np.asarray(ids).reshape(-1)
    keep = (I >= 0) & (I < V) & (I != pad)
    want, size, count = np.zeros((V, D)), np.zeros((V, D)), np.zeros(V)
    np.add.at(want, I[keep], G[keep])
    np.add.at(size, I[keep], np.abs(G[keep]))
    np.add.at(count, I[keep], 1)
    s = float(np.float32(scale))
    bound = (U * (count[:, None] + 2) * size + HALF_STEP[kind] * np.abs(want)) * abs(s) * (1 + 1e-3) + TINY[kind]
    assert tuple(got.shape) == (V, D) and got.dtype == grad.dtype
    ref.check(_f64(got), want * s, bound, what)
    again = ops.embedding_grad(grad, _ids(ids), V, scale=scale, pad_token=pad)
    assert torch.equal(got, again), what + ": two calls differ"
    return got


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (1, 10, 3), (2, 3, 8), (17, 5, 64), (63, 100, 65), (64, 100, 256),
                                   (65, 257, 33), (1000, 300, 100), (1023, 512, 128), (1025, 513, 8), (4000, 10000, 256),
                                   (10241, 1000, 24), (3000, 50001, 40), (5000, 64, 513), (700, 200000, 16)])
def test_embedding_gradient(kind, N, V, D):
    rng = np.random.default_rng(N + V + D)
    grad = _logits(rng, N, D, kind, 1.0)
    _check_embed_grad(grad, rng.integers(0, V, N), V, 1.0, -1, kind, "uniform")
    zipf = np.minimum(rng.zipf(1.3, N) - 1, V - 1)
    _check_embed_grad(grad, zipf, V, 16.0, 0, kind, "by frequency")
    mixed = rng.integers(-3, V + 3, N)
    _check_embed_grad(grad, mixed, V, -0.5, V // 2, kind, "with ids outside")


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("N,V,D", [(5000, 7, 96), (20000, 1000, 256), (40001, 3, 40), (9000, 600, 520), (70000, 50, 16)])
def test_embedding_gradient_of_tokens_that_fill_the_batch(kind, N, V, D):
    """One token in every position, in most, and a few long runs beside short ones."""
    rng = np.random.default_rng(N)
    grad = _logits(rng, N, D, kind, 1.0)
    _check_embed_grad(grad, np.full(N, V - 1), V, 1.0, -1, kind, "one token")
    ids = np.where(rng.random(N) < 0.9, 1, rng.integers(0, V, N))
    _check_embed_grad(grad, ids, V, 0.1, -1, kind, "most")
    runs = np.sort(np.minimum(rng.geometric(0.3, N) - 1, V - 1))[::-1].copy()
    _check_embed_grad(grad, runs, V, 1.0, -1, kind, "runs")
    none = _check_embed_grad(grad, np.full(N, 2), V, 1.0, 2, kind, "all padding")
    assert not none.any()


@pytest.mark.parametrize("N,V,D", [(24576, 300, 8), (24577, 300, 8), (26624, 131072, 4), (26625, 131073, 4), (50000, 1, 3),
                                   (100003, 5000, 12), (300000, 50000, 4)])
def test_embedding_gradient_of_long_batches(N, V, D):
    """Around the length from which the tokens are sorted by way of lists, and the largest table for that."""
    rng = np.random.default_rng(N)
    grad = _logits(rng, N, D, "f32", 1.0)
    _check_embed_grad(grad, rng.integers(-1, V + 1, N), V, 2.0, -1, "f32", "uniform")
    _check_embed_grad(grad, np.minimum(rng.zipf(1.2, N) - 1, V - 1), V, 1.0, 0, "f32", "by frequency")
    _check_embed_grad(grad, np.full(N, V // 2), V, 1.0, -1, "f32", "one token")


def test_embedding_gradient_of_padding_that_holds_nan_and_of_nothing():
    from image_caption_amd import ops
    grad = torch.ones(4, 8, device=dev())
    grad[1] = float("nan")
    got = ops.embedding_grad(grad, _ids([1, 0, 1, 2]), 5, pad_token=0)
    want = torch.zeros(5, 8, device=dev())
    want[1], want[2] = 2.0, 1.0
    assert torch.equal(got, want)
    from image_caption_amd import _lib
    out, ws = torch.ones(5, 8, device=dev()), torch.empty(4096, dtype=torch.uint8, device=dev())
    _lib.call("icap_embedding_grad", grad.data_ptr(), 0, grad.data_ptr(), out.data_ptr(), 0, 5, 8, 1.0, -1,
              ws.data_ptr(), 4096, torch.cuda.current_stream().cuda_stream)      # no tokens at all
    assert not out.any()
    none = ops.embedding_grad(torch.zeros(0, 8, device=dev()), _ids(np.zeros(0)), 5)
    assert tuple(none.shape) == (5, 8) and not none.any()


# ---- together, streams, graphs --------------------------------------------------------------

def _step(ops, w, ids, tokens, tl, ti, adv):
    """A decoder of one dense layer: lookup, logits, policy-gradient and distillation gradients, back
    into the kernel and the table.  Every product runs on the framework's own dense operator."""
    x = ops.embedding_scaled(w["table"], ids, scale=4.0, pad_token=0)
    logits = ops.dense(x, w["kernel"])
    lp, h, stats, top, _ = ops.token_log_probs(logits, tokens, top_k=3, pad_token=0)
    g = ops.token_log_probs_grad(logits, tokens, stats, h, adv, torch.full_like(adv, 0.05), pad_token=0)
    loss, d = ops.distill_loss(logits, tl, ti, 2.0, torch.ones_like(adv))
    g = g + d
    d_kernel = ops.dense(x.t().contiguous(), g)
    d_x = ops.dense(g, w["kernel"].t().contiguous())
    d_table = ops.embedding_grad(d_x, ids, w["table"].shape[0], scale=4.0, pad_token=0)
    return lp, h, top, loss, d_kernel, d_table


def _step_inputs(rng, N=40, V=200, D=16, K=5):
    w = {"table": _dev(rng.standard_normal((V, D)).astype(np.float32) * 0.2),
         "kernel": _dev(rng.standard_normal((D, V)).astype(np.float32) * 0.5)}
    ids, tokens = rng.integers(0, V, N), rng.integers(0, V, N)
    ids[::5] = 0
    tokens[::5] = 0
    ti = np.stack([rng.permutation(V)[:K] for _ in range(N)])
    ti[::5] = -1
    return w, _ids(ids), _ids(tokens), _dev(rng.standard_normal((N, K))), _ids(ti), _dev(rng.standard_normal(N))


def test_a_training_step_of_a_small_decoder():
    """The run of all operators against the same step in float64 with torch's own gradients.  The two
    sides differ by roundings of float32 that two products of 16 and 200 terms pass on: 1e-5 of
    the largest value stands for (16 + 200 + 40) u with a condition of a few units."""
    from image_caption_amd import ops
    rng = np.random.default_rng(0)
    w, ids, tokens, tl, ti, adv = _step_inputs(rng)
    lp, h, top, loss, d_kernel, d_table = _step(ops, w, ids, tokens, tl, ti, adv)
    table, kernel = (w[k].double().cpu().requires_grad_() for k in ("table", "kernel"))
    i, t, q_id = ids.cpu().long(), tokens.cpu().long(), ti.cpu().long()
    live = (t != 0)
    x = table[i] * 4.0 * (i != 0)[:, None]
    z = x @ kernel
    logp = torch.log_softmax(z, -1)
    want_lp = logp.gather(1, t[:, None])[:, 0] * live
    want_h = -(logp.exp() * logp).sum(-1) * live
    q = torch.softmax(tl.double().cpu() / 2.0, -1)
    lt = torch.log_softmax(z / 2.0, -1).gather(1, q_id.clamp_min(0))
    want_loss = 4.0 * (q * (q.log() - lt)).sum(-1) * (q_id[:, 0] >= 0)
    ((adv.double().cpu() * want_lp).sum() + 0.05 * want_h.sum() + want_loss.sum()).backward()
    for name, got, want in (("log_probs", lp, want_lp), ("entropy", h, want_h), ("loss", loss, want_loss),
                            ("kernel", d_kernel, kernel.grad), ("table", d_table, table.grad)):
        want = want.detach().numpy()
        ref.check(_f64(got), want, 1e-5 * np.abs(want).max(), name)
    assert not np_of(d_table)[0].any()


def test_on_another_stream_and_captured():
    """The step on a side stream, and captured into a graph that is replayed with new inputs between
    the program's own work: every replay equals the eager step bit for bit."""
    from image_caption_amd import ops
    rng = np.random.default_rng(1)
    cases = [_step_inputs(rng) for _ in range(3)]
    eager = [_step(ops, *c) for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = _step(ops, *cases[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager[1]))
    hold = [{k: v.clone() for k, v in cases[0][0].items()}] + [v.clone() for v in cases[0][1:]]
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = _step(ops, *hold)
    with torch.cuda.graph(second, stream=side):
        captured2 = _step(ops, *hold)
    for _ in range(2):
        for c, want in zip(cases, eager):
            for k in hold[0]:
                hold[0][k].copy_(c[0][k])
            for a, b in zip(hold[1:], c[1:]):
                a.copy_(b)
            for outs in (captured, captured2):
                for t in outs:
                    t.zero_()
            graph.replay()
            second.replay()
            torch.cuda.synchronize()
            for outs in (captured, captured2):
                assert all(torch.equal(a, b) for a, b in zip(outs, want))
            between = _step(ops, *cases[2])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(between, eager[2]))


def test_refusals_on_the_device():
    from image_caption_amd import _lib, ops
    x, t = torch.zeros(4, 8, device=dev()), _ids(np.zeros(4))
    with pytest.raises(TypeError, match="tokens"):
        ops.token_log_probs(x, t.long())
    with pytest.raises(TypeError, match="logits"):
        ops.token_log_probs(x.double(), t)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_log_probs(x, t.cpu())
    with pytest.raises(ValueError, match="contiguous"):
        ops.token_log_probs(x, torch.zeros(4, 2, dtype=torch.int32, device=dev())[:, 0])
    with pytest.raises(_lib.IcapError, match="token_log_probs"):
        ops.token_log_probs(x[:, :0], t)
    with pytest.raises(_lib.IcapError, match="temperature"):
        ops.distill_loss(x, x[:, :2].contiguous(), _ids(np.zeros((4, 2))), temperature=0.0)
    with pytest.raises(TypeError, match="grad_loss"):
        ops.distill_loss(x, x[:, :2].contiguous(), _ids(np.zeros((4, 2))), grad_loss=t)
    with pytest.raises(ValueError, match="contiguous"):
        ops.embedding_grad(torch.zeros(4, 16, device=dev())[:, ::2], t, 5)
    lp, h, st, top, tlp = ops.token_log_probs(x[:0], t[:0], top_k=2)
    assert lp.shape == (0,) and st.shape == (0, 2) and top.shape == (0, 2)
