"""What torch can ask of the trainer-side operators beside a plain backward pass, as far as it is refused without a GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_tensors_with_a_forward_mode_tangent_are_refused():
    """Their results would have none, which means a derivative of zero.  Refused before anything else is looked at, with and without
    grad mode; where forward mode is off there is nothing to lose."""
    import mpe_hip
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual = lambda *s: fw.make_dual(torch.zeros(*s), torch.ones(*s))
        x, w, b, r = torch.zeros(4, 3), torch.zeros(2, 3), torch.zeros(2), torch.zeros(4, 2)
        p = dict(logits=torch.zeros(4, 5), actions=torch.zeros(4, dtype=torch.int32), old_logp=torch.zeros(4), advantages=torch.zeros(4), values=torch.zeros(4),
                 old_values=torch.zeros(4), returns=torch.zeros(4), weights=torch.zeros(4))
        calls = [lambda: mpe_hip.linear(dual(4, 3), w, b, residual=r), lambda: mpe_hip.linear(x, dual(2, 3)), lambda: mpe_hip.linear(x, w, dual(2)),
                 lambda: mpe_hip.linear(x, w, b, "tanh", dual(4, 2)), lambda: mpe_hip.grad_norm([x, dual(2)]), lambda: mpe_hip.clip_grad_norm([x], 1.0, out=[dual(4, 3)])]
        calls += [lambda k=k: mpe_hip.ppo_loss(**dict(p, **{k: dual(*p[k].shape)})) for k in p if k != "actions"]
        for call in calls:
            for mode in (True, False):
                with torch.set_grad_enabled(mode), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
            with fw._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="GPU"):
                call()


def test_a_clip_below_zero_by_less_than_float32_holds_is_refused():
    from test_learn_cpu import _lib, _ppo
    _, lib = _lib()
    for bad in (-1e-60, -1e-46):
        assert _ppo(lib, clip=bad) == -1 and "clip" in lib.mpe_last_error(None).decode()
