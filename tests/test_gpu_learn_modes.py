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
