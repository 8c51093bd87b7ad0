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


def test_gradient_between_the_rows_of_the_logits_and_over_them():
    from image_caption_amd import ops
    _, t, st, h = _inputs(6)
    buf = torch.zeros(6, 20)
    g = torch.zeros(6)
    # between the rows of the logits: past the check, then refused for not being on the GPU
    for x, out in ((buf[:, :8], buf[:, 8:16]), (buf[:, 12:], buf[:, 2:10]), (buf[:, :8], buf[:, 12:]),
                   (buf[::2, :8], buf[1::2, 4:12])):
        n = len(x)
        with pytest.raises(ValueError, match="GPU"):
            ops.token_log_probs_grad(x, t[:n], st[:n], h[:n], g[:n], out=out)
    cube = buf.view(2, 3, 20)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_log_probs_grad(cube[:, :2, :8], t[:4].view(2, 2), st[:4].view(2, 2, 2), h[:4].view(2, 2),
                                 g[:4].view(2, 2), out=cube[:, 1:, 8:16])
    # over them
    for x, out in ((buf[:, :8], buf[:, 7:15]), (buf[:, 12:], buf[:, 5:13]), (buf[:5, :8], buf[1:, :8]),
                   (buf[:5, 12:], buf.as_strided((5, 8), (18, 1), 30)), (cube[:, :2, :8], cube[:, 1:, :8])):
        shape = x.shape[:-1]
        n = shape.numel()
        with pytest.raises(ValueError, match="overlaps"):
            ops.token_log_probs_grad(x, t[:n].view(shape), st[:n].view(*shape, 2), h[:n].view(shape), g[:n].view(shape),
                                     out=out)


def test_gradient_over_any_other_operand():
    from image_caption_amd import ops
    t, st, h, g = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 2), torch.zeros(4), torch.zeros(4)
    x, pool = torch.zeros(4, 8), torch.zeros(64)
    out = pool[:32].view(4, 8)
    for name, args in (("stats", (pool[24:32].view(4, 2), h, g, g)), ("entropy", (st, pool[31:35], g, g)),
                       ("grad_log_probs", (st, h, pool[:4], g)), ("grad_entropy", (st, h, g, pool[8:12]))):
        for o, y in ((out, x), (out, out)):
            with pytest.raises(ValueError, match="overlaps " + name):
                ops.token_log_probs_grad(y, t, *args, out=o)
    with pytest.raises(ValueError, match="overlaps tokens"):
        ops.token_log_probs_grad(x, pool.view(torch.int32)[4:8], st, h, g, g, out=out)
    tl, ti = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    for name, args in (("teacher_logits", (pool[8:16].view(4, 2), ti, 1.0, g)),
                       ("teacher_ids", (tl, pool.view(torch.int32)[8:16].view(4, 2), 1.0, g)),
                       ("grad_loss", (tl, ti, 1.0, pool[28:32]))):
        with pytest.raises(ValueError, match="overlaps " + name):
            ops.distill_loss(x, *args, out=out)
    with pytest.raises(ValueError, match="GPU"):
        ops.distill_loss(x, tl, ti, 1.0, pool[32:36], out=out)


def test_operands_beside_the_rows_of_a_gradient():
    """Contiguous operands that lie whole behind one of its rows are no part of it."""
    from image_caption_amd import ops
    buf = torch.zeros(4, 40)
    x, t, out = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32), buf[:, 4:12]
    st, h, g = buf[1, 12:20].view(4, 2), buf[0, 30:34], buf[2, 12:16]
    with pytest.raises(ValueError, match="GPU"):
        ops.token_log_probs_grad(x, t, st, h, g, out=out)
    with pytest.raises(ValueError, match="GPU"):
        ops.token_log_probs_grad(buf.view(-1)[92:124].view(4, 8)[:3], t[:3], st[:3], h[:3], g[:3],
                                 out=buf.as_strided((3, 8), (40, 1), 4))
    with pytest.raises(ValueError, match="overlaps stats"):
        ops.token_log_probs_grad(x, t, buf.view(-1)[38:46].view(4, 2), h, g, out=out)
