"""Sizes, inputs and plain forms of the operators a caption decoder is trained with.

Three operators stand between a decoder's two ends and its gradient:

  score / score_grad   log probabilities of given tokens with the entropy of their rows and the
                       best alternatives, and the gradient of the first two (policy gradient,
                       teacher forcing, reporting a caption with its alternatives)
  distill              the loss against a teacher's top logits together with its gradient
  embed / embed_grad   the scaled embedding lookup and its gradient by sorted tokens

`own` selects what `run` calls: the plain torch form of an operator (False) or the framework's
kernels (True).  A case is a dict of plain values; `prepare` makes what a program has in hand
before the call, `run` is one pass, `exact` the same outputs from the definition in 64 bits and
`work` the bytes and operations that a pass cannot do without.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAD, START = 0, 3          # the vocabulary's padding and start tokens: neither is ever a word of a caption


# ---- cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one greedy step of a batch of 32 images, reported with the five best alternatives
        dict(name="score step", op="score", type="f32", N=32, V=10000, ld=10000, k=5, pad=0.0),
        # the captions of 512 images, 20 positions each, scored for a policy gradient
        dict(name="score captions", op="score", type="f32", N=10240, V=10000, ld=10000, k=0, pad=0.25),
        # a large odd vocabulary in bf16 with 16 alternatives: rows that start at every alignment
        dict(name="score wide", op="score", type="bf16", N=2560, V=50001, ld=50001, k=16, pad=0.0),
        # the gradient that follows "score captions"
        dict(name="score captions grad", op="score_grad", type="f32", N=10240, V=10000, ld=10000, pad=0.25),
        # an odd batch over a large odd vocabulary in fp16, rows of a padded logits buffer
        dict(name="score wide grad", op="score_grad", type="f16", N=1271, V=50001, ld=50048, pad=0.1),
        # a small batch against a teacher that hands over 8 logits a position, 5000-word vocabulary
        dict(name="distill step", op="distill", type="f32", N=64, V=5000, ld=5000, K=8, temperature=1.0, pad=0.0),
        # a training batch: 512 captions of 20 positions, 20 teacher logits
        dict(name="distill captions", op="distill", type="f32", N=10240, V=10000, ld=10000, K=20,
             temperature=2.0, pad=0.25),
        # a large vocabulary in bf16, 64 teacher logits
        dict(name="distill wide", op="distill", type="bf16", N=2048, V=50000, ld=50000, K=64,
             temperature=2.0, pad=0.1),
        # the lookup of one beam step: 32 images, beam 3
        dict(name="embed step", op="embed", type="f32", N=96, V=10000, D=256, pad=0.0),
        # the lookup of a long batch out of a large bf16 table
        dict(name="embed batch", op="embed", type="bf16", N=131072, V=50000, D=512, pad=0.1),
        # its gradient for 512 captions of 20 words, word frequencies falling with their rank
        dict(name="embed captions grad", op="embed_grad", type="f32", N=10240, V=10000, D=256, pad=0.25),
        # and for a long batch over a large vocabulary
        dict(name="embed batch grad", op="embed_grad", type="bf16", N=131071, V=50000, D=512, pad=0.1),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score_grad", "distill", "embed", "embed_grad"])
    case = dict(op=op, type=rng.choice(sorted(TYPES)))
    if op in ("embed", "embed_grad"):
        case.update(N=_log_uniform(rng, 1, 131072), V=_log_uniform(rng, 64, 50000))
        case.update(D=rng.choice([_log_uniform(rng, 8, 512), 8 * rng.randint(4, 64)]))
    else:
        V = _log_uniform(rng, 200, 131072)
        N = _log_uniform(rng, 1, max(2, min(16384, 100_000_000 // V)))
        case.update(N=N, V=V, ld=V + rng.choice([0, 0, -V % 64, rng.randint(1, 40)]))
    if op == "score":
        case.update(k=rng.choice([0, 1, 5, rng.randint(2, 32)]))
    if op == "distill":
        case.update(K=_log_uniform(rng, 1, 128), temperature=rng.choice([1.0, 2.0, round(rng.uniform(0.5, 4.0), 2)]))
    case.update(pad=rng.choice([0.0, 0.1, 0.25]))
    return case


# ---- inputs --------------------------------------------------------------------------------

def _padded(case):
    """Rows (or tokens) of the case that are padding."""
    return int(case["N"] * case["pad"])


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _frequencies(V):
    """Word frequencies falling with the rank, as a fitted vocabulary's do (on the host, so that every call gives the same)."""
    p = 1.0 / (torch.arange(V, dtype=torch.float64) + 3.0)
    p[PAD] = 0.0
    p[START] = 0.0
    return p / p.sum()


def _tokens(case, g):
    V, N = case["V"], case["N"]
    up_to = torch.cumsum(_frequencies(V), 0).cuda()
    t = torch.searchsorted(up_to, torch.rand(N, device="cuda", dtype=torch.float64, generator=g), right=True)
    t = t.clamp_max(V - 1).to(torch.int32)
    t[torch.randperm(N, device="cuda", generator=g)[:_padded(case)]] = PAD
    return t


def _logits(case, g):
    """Rows of a decoder: a bias by word frequency, a spread of some units, the pad and start columns masked."""
    N, V, t = case["N"], case["V"], TYPES[case["type"]]
    x = torch.randn(N, V, device="cuda", generator=g)
    x.mul_(2.0).add_(torch.log(_frequencies(V).clamp_min(1e-9)).float().cuda() * 0.5)
    x[:, START] = -math.inf if case["type"] == "f16" else torch.finfo(t).min
    x[:, PAD] = -math.inf
    buf = torch.zeros(N, case["ld"], device="cuda", dtype=t)
    buf[:, :V] = x
    return buf[:, :V]


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    op, N, V = case["op"], case["N"], case["V"]
    if op in ("embed", "embed_grad"):
        s["ids"] = _tokens(case, g)
        s["scale"] = math.sqrt(case["D"])
        shape = (V if op == "embed" else N, case["D"])
        spread = 0.05 if op == "embed" else 1.0
        s["table" if op == "embed" else "grad"] = (torch.randn(*shape, device="cuda", generator=g) * spread).to(TYPES[case["type"]])
        return s
    s["logits"] = x = _logits(case, g)
    if op == "distill":
        # the teacher sees the same rows a little differently and hands over its K best
        K = min(case["K"], V)
        best, ids = torch.topk(x.float() + torch.randn(N, V, device="cuda", generator=g), K, dim=-1)
        ids = ids.to(torch.int32)
        ids[torch.randperm(N, device="cuda", generator=g)[:_padded(case)]] = -1
        ids[torch.rand(N, device="cuda", generator=g) < 0.1, K // 2 + 1:] = -1        # shorter lists
        s["teacher_logits"], s["teacher_ids"] = best.to(x.dtype), ids
        s["grad_loss"] = torch.rand(N, device="cuda", generator=g) + 0.5
        return s
    s["tokens"] = _tokens(case, g)
    if op == "score_grad":
        _, s["entropy"], s["stats"] = _plain_score(x, s["tokens"])
        s["grad_log_probs"] = torch.randn(N, device="cuda", generator=g)
        s["grad_entropy"] = torch.full((N,), -0.01, device="cuda")
    return s


# ---- plain forms ---------------------------------------------------------------------------

def _plain_score(x, tokens):
    """(log probability of the token, entropy, (row maximum, log of the sum of exponentials)); rows of PAD tokens give 0."""
    x = x.float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    s = e.sum(-1)
    log_s = torch.log(s)
    entropy = log_s - torch.where(e > 0, e * d, 0.0).sum(-1) / s
    lp = d.gather(1, tokens.long()[:, None])[:, 0] - log_s
    live = tokens != PAD
    stats = torch.stack([m[:, 0], log_s], -1)
    return lp.where(live, 0.0), entropy.where(live, 0.0), stats.where(live[:, None], 0.0)


def _plain_top(x, tokens, stats, k):
    """The k largest logits of each row, ties to the lowest index: one 64-bit key of value and index for each."""
    i = (x.float() + 0.0).view(torch.int32)
    key = torch.where(i < 0, i ^ 0x7FFFFFFF, i).long() << 32
    key += torch.arange(x.shape[1] - 1, -1, -1, device=x.device)
    ids = x.shape[1] - 1 - (torch.topk(key, k, dim=-1).values & 0xFFFFFFFF)
    lp = x.float().gather(1, ids) - stats[:, :1] - stats[:, 1:]
    live = (tokens != PAD)[:, None]
    return ids.where(live, -1).to(torch.int32), lp.where(live, 0.0)


def _plain_score_grad(x, tokens, stats, entropy, g_lp, g_h):
    lp = x.float() - stats[:, :1] - stats[:, 1:]
    p = torch.exp(lp)
    g = -g_lp[:, None] * p - g_h[:, None] * torch.where(p > 0, p * (lp + entropy[:, None]), 0.0)
    g.scatter_add_(1, tokens.long()[:, None], g_lp[:, None])
    return g.where((tokens != PAD)[:, None], 0.0).to(x.dtype)


def _plain_distill(x, t_logits, t_ids, temperature, g_loss):
    there = t_ids >= 0
    at = t_ids.clamp_min(0).long()
    t = torch.where(there, t_logits.float(), -math.inf) / temperature
    live = there.any(-1)
    t = t - t.amax(-1, keepdim=True).where(live[:, None], 0.0)
    log_q = t - torch.log(torch.exp(t).sum(-1, keepdim=True))
    q = torch.exp(log_q).where(there, 0.0)
    d = (x.float() - x.float().amax(-1, keepdim=True)) / temperature
    lp = d - torch.log(torch.exp(d).sum(-1, keepdim=True))
    loss = temperature ** 2 * torch.where(q > 0, q * (log_q - lp.gather(1, at)), 0.0).sum(-1)
    g = torch.exp(lp)
    g.scatter_add_(1, at, -q)
    g = g * (g_loss * temperature)[:, None]
    return loss.where(live, 0.0), g.where(live[:, None], 0.0).to(x.dtype)


def _plain_embed(table, ids, scale):
    return (table[ids.long()].float() * scale).where((ids != PAD)[:, None], 0.0).to(table.dtype)


def _plain_embed_grad(grad, ids, V, scale):
    g = (grad.float() * scale).where((ids != PAD)[:, None], 0.0)
    return torch.zeros(V, grad.shape[1], device=grad.device).index_add_(0, ids.long(), g).to(grad.dtype)


def run(s):
    if own:
        return _own(s)
    op = s["op"]
    if op == "score":
        lp, entropy, stats = _plain_score(s["logits"], s["tokens"])
        top = _plain_top(s["logits"], s["tokens"], stats, s["k"]) if s["k"] else ()
        return (lp, entropy, stats, *top)
    if op == "score_grad":
        return _plain_score_grad(s["logits"], s["tokens"], s["stats"], s["entropy"], s["grad_log_probs"], s["grad_entropy"])
    if op == "distill":
        return _plain_distill(s["logits"], s["teacher_logits"], s["teacher_ids"], s["temperature"], s["grad_loss"])
    if op == "embed":
        return _plain_embed(s["table"], s["ids"], s["scale"])
    return _plain_embed_grad(s["grad"], s["ids"], s["V"], s["scale"])


# ---- the framework's calls -----------------------------------------------------------------

def _own(s):
    from image_caption_amd import ops
    op = s["op"]
    if op == "score":
        out = ops.token_log_probs(s["logits"], s["tokens"], top_k=s["k"], pad_token=PAD)
        return out if s["k"] else out[:3]
    if op == "score_grad":
        return ops.token_log_probs_grad(s["logits"], s["tokens"], s["stats"], s["entropy"],
                                        grad_log_probs=s["grad_log_probs"], grad_entropy=s["grad_entropy"],
                                        pad_token=PAD)
    if op == "distill":
        return ops.distill_loss(s["logits"], s["teacher_logits"], s["teacher_ids"],
                                temperature=s["temperature"], grad_loss=s["grad_loss"])
    if op == "embed":
        return ops.embedding_scaled(s["table"], s["ids"], scale=s["scale"], pad_token=PAD)
    return ops.embedding_grad(s["grad"], s["ids"], s["V"], scale=s["scale"], pad_token=PAD)


# ---- what a pass cannot do without ---------------------------------------------------------

def work(case):
    size = 4 if case["type"] == "f32" else 2
    op, N, V = case["op"], case["N"], case["V"]
    live = N - _padded(case)
    if op == "embed":
        # distinct rows are read once: a batch meets at most V of them
        D = case["D"]
        return {"bytes": N * 4 + (min(live, V) + N) * D * size, "flops": live * D}
    if op == "embed_grad":
        D = case["D"]
        return {"bytes": N * 4 + (live + V) * D * size, "flops": (live + V) * D}
    if op == "score":
        return {"bytes": live * V * size + N * (4 + 16 + 8 * case["k"]), "flops": 6 * live * V}
    if op == "score_grad":
        return {"bytes": (live + N) * V * size + N * 24, "flops": 8 * live * V}
    return {"bytes": (live + N) * V * size + N * (8 + case["K"] * (4 + size)), "flops": 8 * live * V}


# ---- the definitions in 64 bits ------------------------------------------------------------

def _exact_rows(x, temperature=1.0):
    """(log probabilities, entropies, maxima, logs of the sums) of float64 rows."""
    z = x.double() / temperature
    lse = torch.logsumexp(z, -1)
    lp = z - lse[:, None]
    h = -torch.special.xlogy(lp.exp(), lp.exp()).sum(-1)
    return lp, h, z.max(-1).values, lse


def exact(case, seed):
    s = prepare(case, seed)
    op, N = s["op"], s["N"]
    if op == "embed":
        rows = s["table"].double().index_select(0, s["ids"].long()) * s["scale"]
        rows[s["ids"] == PAD] = 0
        return rows
    if op == "embed_grad":
        out = torch.zeros(s["V"], s["D"], dtype=torch.float64, device="cuda")
        keep = (s["ids"] != PAD).nonzero()[:, 0]
        out.index_add_(0, s["ids"][keep].long(), s["grad"][keep].double())
        return out * s["scale"]
    parts = []
    for lo in range(0, N, 512):
        r = slice(lo, min(lo + 512, N))
        x = s["logits"][r]
        if op == "distill":
            tau, ids = s["temperature"], s["teacher_ids"][r].long()
            dead = (ids < 0).all(-1)
            log_q = torch.log_softmax((s["teacher_logits"][r].double() / tau).masked_fill(ids < 0, -math.inf), -1)
            q = log_q.exp().masked_fill(ids < 0, 0.0)
            lp = _exact_rows(x, tau)[0]
            picked = lp.gather(1, ids.clamp_min(0))
            loss = tau * tau * (torch.special.xlogy(q, q) - torch.where(q > 0, q * picked, 0.0)).sum(-1)
            g = lp.exp().scatter_add(1, ids.clamp_min(0), -q) * (tau * s["grad_loss"][r].double())[:, None]
            parts.append((loss.masked_fill(dead, 0.0), g.masked_fill(dead[:, None], 0.0)))
            continue
        t = s["tokens"][r].long()
        dead = t == PAD
        lp, h, top, lse = _exact_rows(x)
        if op == "score":
            stats = torch.stack([top, lse - top], -1).masked_fill(dead[:, None], 0.0)
            got = (lp.gather(1, t[:, None])[:, 0].masked_fill(dead, 0.0), h.masked_fill(dead, 0.0), stats)
            if s["k"]:
                got += (lp.topk(s["k"], -1).values.masked_fill(dead[:, None], 0.0),)
            parts.append(got)
            continue
        p = lp.exp()
        one = torch.nn.functional.one_hot(t, x.shape[1]).double()
        g = s["grad_log_probs"][r].double()[:, None] * (one - p)
        g -= s["grad_entropy"][r].double()[:, None] * (torch.special.xlogy(p, p) + p * h[:, None])
        parts.append((g.masked_fill(dead[:, None], 0.0),))
    out = [torch.cat(v) for v in zip(*parts)]
    if op == "score" and s["k"]:
        return (*out[:3], None, out[3])      # the alternatives' ids are whole numbers
    return out[0] if op == "score_grad" else tuple(out)
