"""Views whose memory does not hold their values: the feed-forward operators read memory, so they refuse them."""
import pytest
import torch


def column(rows, device="cpu"):
    """-1s in a view with a pending negation whose strides are a matrix' own: the imaginary part of a conjugate."""
    t = torch.complex(torch.zeros(rows, 1, device=device), torch.ones(rows, 1, device=device)).conj().imag
    assert t.is_neg() and t.shape == (rows, 1)
    return t


def test_a_pending_negation_is_refused():
    from fpn import feed_forward as F
    x, w = column(4), torch.ones(1, 16)
    for call in (lambda: F._first("x", x), lambda: F._tensor("x", x, x, (4, 1)), lambda: F._kept("x", x, x, (4, 1)), lambda: F.dense(x, w),
                 lambda: F.gated(x, w, w), lambda: F.gated_feed_forward(x, w, w, w.t()), lambda: F.gated_grad(x, x, w, w, x, x)):
        with pytest.raises(ValueError, match="x has a pending negation"):
            call()
    with pytest.raises(ValueError, match="ROCm device"):
        F.dense(x.resolve_neg(), w)


@pytest.mark.gpu
def test_a_pending_negation_is_refused_on_the_device(device):
    from fpn import feed_forward as F
    x, w, n = torch.ones(4, 8, device=device), torch.ones(1, 16, device=device), column(4, device)
    with pytest.raises(ValueError, match="x has a pending negation"):
        F.dense(n, w)
    with pytest.raises(ValueError, match="w has a pending negation"):
        F.dense(x, column(8, device))
    with pytest.raises(ValueError, match="residual has a pending negation"):
        F.dense(x, torch.ones(8, 1, device=device), residual=n)
    assert (F.dense(n.resolve_neg(), w) == -1).all()


@pytest.mark.gpu
def test_a_negated_gradient_is_taken_as_what_it_says(device):
    from fpn import feed_forward as F
    x = torch.randn((4, 8), generator=torch.Generator().manual_seed(1)).to(device).requires_grad_()
    w, r = torch.ones((8, 1), device=device), torch.zeros((4, 1), device=device, requires_grad=True)
    for act in (None, "gelu"):
        y = F.dense(x, w, None, act, r)
        got = torch.autograd.grad(y, (x, r), column(4, device), retain_graph=True)
        want = torch.autograd.grad(y, (x, r), -torch.ones((4, 1), device=device))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
