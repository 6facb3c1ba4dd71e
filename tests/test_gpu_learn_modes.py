"""What torch can ask of the trainer-side operators beside a plain backward pass: refused, not answered wrongly."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_forward_mode_is_refused_in_every_operator_and_backward_pass():
    import mpe_hip
    import torch.autograd.forward_ad as fw
    x, w = torch.randn(4, 3, device=DEV), torch.randn(2, 3, device=DEV, requires_grad=True)
    y = mpe_hip.linear(x, w, None, "tanh")
    logits = torch.randn(4, 5, device=DEV, requires_grad=True)
    loss, _ = mpe_hip.ppo_loss(logits, torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(4, device=DEV), torch.ones(4, device=DEV))
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for mode in (True, False):
            with torch.set_grad_enabled(mode), pytest.raises(NotImplementedError, match="forward-mode"):
                mpe_hip.linear(d, w)
        for out, leaf in ((y, w), (loss, logits)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaf, fw.make_dual(torch.ones_like(out), torch.ones_like(out)), retain_graph=True)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            mpe_hip.grad_norm([d])
    assert torch.equal(mpe_hip.linear(x, w.detach(), None, "tanh"), y.detach()) and torch.autograd.grad(y, w, torch.ones_like(y))[0].shape == w.shape


@pytest.mark.parametrize("transform", ["jvp", "grad", "vmap"])
def test_function_transforms_are_refused(transform):
    """Their tensors are wrappers without memory of their own."""
    import mpe_hip
    x, w = torch.randn(4, 3, device=DEV), torch.randn(2, 3, device=DEV)
    f = lambda t: mpe_hip.linear(t, w).sum()
    with pytest.raises(RuntimeError):
        if transform == "jvp":
            torch.func.jvp(f, (x,), (torch.ones_like(x),))
        elif transform == "grad":
            torch.func.grad(f)(x)
        else:
            torch.func.vmap(f)(x[:, None])


def test_views_of_the_negative_of_their_memory():
    """The imaginary part of a conjugate: torch keeps the sign as a mark on the tensor."""
    import mpe_hip
    neg = lambda *s: torch.randn(*s, dtype=torch.complex64, device=DEV).conj().imag
    plain = lambda t: torch.empty_like(t).copy_(t)
    x, w, b, dy = neg(40, 1), neg(3, 1), neg(3), neg(40, 3)
    assert x.is_neg() and w.is_neg() and not plain(x).is_neg()
    for first in ((x, w, b, dy), (torch._neg_view(plain(x)), torch._neg_view(plain(w)), torch._neg_view(plain(b)), torch._neg_view(plain(dy))),
                  (neg(1, 40), neg(30, 40), neg(30), neg(1, 30))):
        got, want = [], []
        for out, q in ((got, first), (want, [plain(t) for t in first])):
            leaves = [t.requires_grad_(True) for t in q[:3]]
            y = mpe_hip.linear(*leaves, "tanh")
            out += [y.detach()] + list(torch.autograd.grad(y, leaves, q[3]))
        assert all(torch.equal(p, q) for p, q in zip(got, want))
    logits, act = torch._neg_view(torch.randn(6, 5, device=DEV)), torch.zeros(6, dtype=torch.int32, device=DEV)
    rest = [torch._neg_view(torch.randn(6, device=DEV)) for _ in range(5)]
    one, two = (mpe_hip.ppo_loss(f(logits), act, *[f(t) for t in rest], weights=f(rest[0])) for f in (lambda t: t, plain))
    assert torch.equal(one[0], two[0]) and torch.equal(one[1], two[1])
    for bad in (torch._neg_view(torch.randn(4, device=DEV)), neg(1)):
        with pytest.raises(ValueError, match="negative view"):
            mpe_hip.grad_norm([bad])
        with pytest.raises(ValueError, match="out 0"):
            mpe_hip.clip_grad_norm([plain(bad)], 1.0, out=[bad])
