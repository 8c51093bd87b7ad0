"""Float64 restatement of the operators that score tokens, with the error bounds their tests use.

A bound counts roundings: u = 2^-24 is half a step of float32, and a sum of n terms whose parts
join in any order is off by at most n * u of the sum of the magnitudes."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}      # smallest subnormals


def sum_terms(V):
    """Roundings a row's sum can go through: the elements of the busiest lane of the narrowest
    workgroup (64 lanes) one after another, and 24 joins of parts with a product each."""
    return V / 64 + 8 + 3 * 24


def softmax_rows(x, tau=1.0):
    """(log p, p, m, log s, none) of float64 rows; a row of -inf alone is `none`."""
    m = np.max(np.where(np.isnan(x), -np.inf, x), axis=-1, keepdims=True)
    none = np.isneginf(x).all(-1)
    with np.errstate(all="ignore"):
        d = (x - m) / tau
        s = np.exp(d).sum(-1, keepdims=True)
        lp = d - np.log(s)
    return lp, np.exp(lp), m[..., 0], np.log(s)[..., 0], none


def score(x, tokens, pad, k):
    """x [N,V] float64 -> log_probs, entropy, stats, top_ids, top_log_probs."""
    N, V = x.shape
    lp, p, m, log_s, none = softmax_rows(x)
    with np.errstate(all="ignore"):
        h = -np.where(p > 0, p * lp, np.where(np.isnan(p), np.nan, 0.0)).sum(-1)
    out, stats = np.empty(N), np.stack([m, log_s], -1)
    for n in range(N):
        t = int(tokens[n])
        out[n] = lp[n, t] if 0 <= t < V else np.nan
        if none[n]:
            out[n] = -np.inf if 0 <= t < V else np.nan
            h[n], stats[n] = 0.0, (-np.inf, 0.0)
    ids = np.empty((N, k), np.int64)
    top = np.empty((N, k))
    for n in range(N):
        v = np.where(np.isnan(x[n]), -np.inf, x[n]) + 0.0
        ids[n] = np.lexsort((np.arange(V), -v))[:k]
        top[n] = -np.inf if none[n] else lp[n, ids[n]]
    gone = tokens == pad
    out[gone], h[gone], stats[gone], ids[gone], top[gone] = 0, 0, 0, -1, 0
    return out, h, stats, ids, top


def score_grad(x, tokens, pad, g_lp, g_h):
    N, V = x.shape
    lp, p, _, _, none = softmax_rows(x)
    with np.errstate(all="ignore"):
        plp = np.where(p > 0, p * lp, np.where(np.isnan(p), np.nan, 0.0))
        h = -plp.sum(-1, keepdims=True)
        g = -g_lp[:, None] * p - g_h[:, None] * (plp + p * h)
    for n in range(N):
        t = int(tokens[n])
        if 0 <= t < V:
            g[n, t] += g_lp[n]
        elif g_lp[n] != 0:
            g[n] = np.nan
        if t == pad or none[n] or (g_lp[n] == 0 and g_h[n] == 0):
            g[n] = 0
    return g


def distill(x, t_logits, t_ids, tau, g_loss=None):
    """(loss [N], gradient [N,V] or None)."""
    N, V = x.shape
    lp, p, _, _, none = softmax_rows(x, tau)
    loss, g = np.empty(N), np.zeros((N, V))
    for n in range(N):
        at = [(int(i), float(t)) for i, t in zip(t_ids[n], t_logits[n]) if int(i) != -1 and not np.isneginf(t)]
        if any(int(i) != -1 and not 0 <= int(i) < V for i in t_ids[n]):
            loss[n] = np.nan
            g[n] = np.nan if g_loss is not None and g_loss[n] != 0 else 0.0
            continue
        if not at:
            loss[n] = 0.0
            continue
        t = np.array([v for _, v in at]) / tau
        with np.errstate(all="ignore"):
            log_q = t - np.max(t)
            log_q -= np.log(np.exp(log_q).sum())
            q = np.exp(log_q)
        if none[n]:
            loss[n] = np.inf
            continue
        with np.errstate(all="ignore"):
            terms = [qi * (lqi - lp[n, i]) for (i, _), qi, lqi in zip(at, q, log_q) if not qi == 0.0]
        loss[n] = tau * tau * np.sum(terms)
        if g_loss is not None and g_loss[n] != 0:
            g[n] = p[n]
            for (i, _), qi in zip(at, q):
                g[n, i] -= qi
            g[n] *= g_loss[n] * tau
    return loss, (g if g_loss is not None else None)


def check(got, ref, bound, what=""):
    """|got - ref| <= bound elementwise; NaN and infinities at the same places."""
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    bound = np.broadcast_to(bound, ref.shape)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(ref), err_msg=what + ": NaN")
    inf = np.isinf(ref)
    np.testing.assert_array_equal(got[inf], ref[inf], err_msg=what + ": infinities")
    fin = np.isfinite(ref)
    assert np.isfinite(got[fin]).all(), what + ": infinite where it should not be"
    d = np.abs(got[fin] - ref[fin])
    bad = (d != 0) & ~(d <= bound[fin])      # (a row of zeros has no bound to speak of where it held NaN)
    assert not bad.any(), "%s: %d of %d off, worst %.3g where %.3g is allowed" % (
        what, bad.sum(), bad.size, d[bad].max(), bound[fin][bad][np.argmax(d[bad])])


def row_bounds(x, tau=1.0):
    """Per row: the relative error that s = sum exp((x - m) / tau) can have, and the magnitude
    D = sum p |x - m| / tau that its exponents' errors and w come from.  One exponential: the
    difference, its product with the rate and the rate's own rounding are three relative errors
    of the exponent, which act with its size; the instruction itself adds two."""
    lp, p, m, log_s, none = softmax_rows(x, tau)
    with np.errstate(all="ignore"):
        D = np.where(p > 0, p * np.abs(x - m[:, None]) / tau, 0.0).sum(-1)
    return U * (sum_terms(x.shape[1]) + 3 * 1.5 * D + 2), D, log_s
