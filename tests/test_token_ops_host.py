"""What the operators that score tokens refuse, checked on the host before anything is launched."""
import ctypes as C

import numpy as np
import pytest
import torch

from tests import token_reference as ref

P = C.c_void_p(64)      # stands for a device pointer; the host never follows it


def _lib():
    from image_caption_amd import _lib
    return _lib, _lib.load()


def _score(lib, logits=P, dtype=0, N=4, V=8, inner=4, ld=8, outer=0, tokens=P, pad=-1, k=0, lp=P, h=P, st=P,
           ids=None, top=None):
    return lib.icap_token_log_probs(logits, dtype, N, V, inner, ld, outer, tokens, pad, k, lp, h, st, ids, top, None)


def _score_grad(lib, logits=P, dtype=0, N=4, V=8, inner=4, ld=8, outer=0, tokens=P, st=P, h=P, out=P, out_ld=8,
                out_outer=0):
    return lib.icap_token_log_probs_grad(logits, dtype, N, V, inner, ld, outer, tokens, -1, st, h, None, None, out,
                                         out_ld, out_outer, None)


def _distill(lib, logits=P, dtype=0, N=4, V=8, inner=4, ld=8, outer=0, tl=P, td=0, ti=P, K=3, tau=1.0, g=P, loss=P,
             out=P, out_ld=8, out_outer=0):
    return lib.icap_distill_loss(logits, dtype, N, V, inner, ld, outer, tl, td, ti, K, tau, g, loss, out, out_ld,
                                 out_outer, None)


@pytest.mark.parametrize("bad", [dict(logits=None), dict(tokens=None), dict(lp=None), dict(h=None), dict(st=None),
                                 dict(dtype=3), dict(dtype=-1), dict(N=0), dict(N=-1), dict(V=0), dict(inner=0),
                                 dict(ld=-1), dict(outer=-8), dict(k=-1), dict(k=9, ids=P, top=P), dict(k=2),
                                 dict(k=2, ids=P)])
def test_token_log_probs_refuses(bad):
    mod, lib = _lib()
    assert _score(lib, **bad) == -1
    assert "token_log_probs" in mod.last_error()


def test_limits_of_alternatives_and_teacher_entries():
    mod, lib = _lib()
    assert _score(lib, V=100, ld=100, k=mod.MAX_ALTERNATIVES + 1, ids=P, top=P) == -3
    assert _distill(lib, K=mod.MAX_TEACHER_LOGITS + 1) == -3
    most = 1 << 30
    assert _score(lib, N=most + 1, V=1, ld=1, inner=most + 1) == -3
    assert _score_grad(lib, N=most + 1, V=1, ld=1, inner=most + 1, out_ld=1) == -3
    assert _score_grad(lib, N=most, V=8192, ld=8192, inner=most, out_ld=8192) == -3
    assert _distill(lib, N=most + 1, V=1, ld=1, inner=most + 1, out_ld=1) == -3
    assert _score(lib, N=1, V=most + 1, ld=most + 1) == -3
    assert lib.icap_embedding_scaled(P, 0, P, P, (1 << 25) + 1, 8, 8, 1.0, -1, None) == -3
    assert lib.icap_embedding_grad(P, 0, P, P, 8, (1 << 25) + 1, 8, 1.0, -1, P, 1 << 40, None) == -3


@pytest.mark.parametrize("bad", [dict(logits=None), dict(tokens=None), dict(st=None), dict(h=None), dict(out=None),
                                 dict(dtype=7), dict(N=0), dict(V=0), dict(out_ld=7), dict(out_ld=0),
                                 dict(inner=2, out_ld=8, out_outer=8), dict(inner=2, out_ld=8, out_outer=15),
                                 dict(inner=2, out_ld=15, out_outer=8), dict(inner=1, out_ld=0, out_outer=4)])
def test_token_log_probs_grad_refuses(bad):
    _, lib = _lib()
    assert _score_grad(lib, **bad) == -1


@pytest.mark.parametrize("bad", [dict(logits=None), dict(tl=None), dict(ti=None), dict(loss=None), dict(K=0),
                                 dict(dtype=3), dict(td=5), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("nan")),
                                 dict(tau=float("inf")), dict(g=None), dict(out=None), dict(out_ld=5), dict(N=0)])
def test_distill_loss_refuses(bad):
    _, lib = _lib()
    assert _distill(lib, **bad) == -1


def test_embedding_entry_points_refuse():
    mod, lib = _lib()
    size = lib.icap_embedding_grad_workspace_bytes(10, 20, 4)
    assert size > 0 and lib.icap_embedding_grad_workspace_bytes(10, 0, 4) == 0
    assert lib.icap_embedding_grad_workspace_bytes(-1, 5, 4) == 0
    for bad in ((None, 0, P, P, 10, 20, 4), (P, 0, None, P, 10, 20, 4), (P, 0, P, None, 10, 20, 4),
                (P, 3, P, P, 10, 20, 4), (P, 0, P, P, 10, 0, 4), (P, 0, P, P, 10, 20, 0), (P, 0, P, P, -1, 20, 4)):
        assert lib.icap_embedding_scaled(*bad, 1.0, -1, None) == -1
        assert lib.icap_embedding_grad(*bad, 1.0, -1, P, 1 << 20, None) == -1
    ok = (P, 0, P, P, 10, 20, 4, 1.0, -1)
    assert lib.icap_embedding_grad(*ok, None, size, None) == -1
    assert lib.icap_embedding_grad(*ok, P, size - 1, None) == -1
    assert lib.icap_embedding_grad(*ok, C.c_void_p(68), size, None) == -1
    assert "workspace" in mod.last_error()


def test_python_front_end_refuses_on_the_host():
    from image_caption_amd import ops
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_log_probs(x, t)
    with pytest.raises(ValueError, match=r"\[..., V\]"):
        ops.token_log_probs(x, t[:3])
    with pytest.raises(ValueError, match="top_k"):
        ops.token_log_probs(x, t, top_k=9)
    with pytest.raises(ValueError, match="top_k"):
        ops.token_log_probs(torch.zeros(4, 100), t, top_k=33)
    st, h = torch.zeros(4, 2), torch.zeros(4)
    with pytest.raises(ValueError, match="stats"):
        ops.token_log_probs_grad(x, t, st[:3], h)
    with pytest.raises(ValueError, match="shape"):
        ops.token_log_probs_grad(x, t, st, h, grad_log_probs=torch.zeros(3))
    with pytest.raises(ValueError, match="shape and dtype"):
        ops.token_log_probs_grad(x, t, st, h, h, out=torch.zeros(4, 9))
    buf = torch.zeros(5 * 8)
    with pytest.raises(ValueError, match="overlaps"):
        ops.token_log_probs_grad(buf[:32].view(4, 8), t, st, h, h, out=buf[8:].view(4, 8))
    ids = torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="teacher"):
        ops.distill_loss(x, torch.zeros(4, 2), ids)
    with pytest.raises(ValueError, match="teacher"):
        ops.distill_loss(x, torch.zeros(4, 0), ids[:, :0])
    with pytest.raises(ValueError, match="one value per row"):
        ops.distill_loss(x, torch.zeros(4, 3), ids, grad_loss=torch.zeros(5))
    with pytest.raises(ValueError, match="out needs"):
        ops.distill_loss(x, torch.zeros(4, 3), ids, out=x)
    with pytest.raises(ValueError, match="ids"):
        ops.embedding_grad(torch.zeros(4, 8), t[:3], 10)
    with pytest.raises(ValueError, match="vocab_size"):
        ops.embedding_grad(torch.zeros(4, 8), t, 0)
    with pytest.raises(ValueError, match="GPU"):
        ops.embedding_scaled(x, t)


def test_row_splits_of_views():
    from image_caption_amd import ops
    x = torch.zeros(3, 5, 8)
    assert ops._row_split(x, "x")[:2] == (15, 8)
    assert ops._row_split(x[:, :-1], "x") == (4, 8, 40)
    assert ops._row_split(x.transpose(0, 1), "x") == (3, 40, 8)
    assert ops._row_split(torch.zeros(4, 10)[:, :7], "x") == (4, 10, 0)
    assert ops._row_strides(x[:, :-1], torch.zeros(3, 4, 8)) == (4, 8, 40, 8, 32)
    assert ops._row_strides(torch.zeros(3, 4, 8), x[:, :-1]) == (4, 8, 32, 8, 40)
    with pytest.raises(ValueError, match="apart"):
        ops._row_split(torch.zeros(2, 3, 5, 8)[:, :, 1:], "x")


def _differences(f, x, step=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        y = x.copy()
        y[i] += step
        up = f(y)
        y[i] -= 2 * step
        g[i] = (up - f(y)) / (2 * step)
    return g


def test_reference_gradients_are_the_differences_of_the_reference():
    """The formulas that the kernels are held to, against central differences (error: step^2 of the
    third derivatives and 2^-53 / step of rounding, together under 1e-8 here)."""
    rng = np.random.default_rng(0)
    x, t = rng.standard_normal((3, 6)), np.array([2, 0, 5])
    gl, gh = rng.standard_normal(3), rng.standard_normal(3)

    def total(y):
        lp, h, *_ = ref.score(y, t, -1, 0)
        return (gl * lp + gh * h).sum()
    np.testing.assert_allclose(ref.score_grad(x, t, -1, gl, gh), _differences(total, x), atol=1e-8)
    tl, ti = rng.standard_normal((3, 4)), np.array([[0, 2, 5, 1], [3, 3, -1, 0], [4, 1, 1, 1]])

    def loss(y):
        return (gl * ref.distill(y, tl, ti, 1.7)[0]).sum()
    np.testing.assert_allclose(ref.distill(x, tl, ti, 1.7, gl)[1], _differences(loss, x), atol=1e-8)
