"""The trainer-side operators as they are used: a rollout of the batched worlds, advantages, the policy's layers, the loss, its
gradients through every layer, clipping, and a step; against the same update written in float64."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _collect(B=64, T=12):
    import mpe_hip
    venv = mpe_hip.BatchedVecEnv("simple_spread", B, max_episode_steps=6, seed=11)
    A = venv.n_agents
    obs = venv.reset()
    gen = torch.Generator(DEV).manual_seed(2)
    O, R, D, ACT = [], [], [], []
    for _ in range(T):
        O.append(obs.view(B, A, -1).clone())
        act = torch.randint(0, 5, (B, A), dtype=torch.int32, device=DEV, generator=gen)
        obs, rew, done, _ = venv.step(act)
        ACT.append(act)
        R.append(rew.clone())
        D.append(done.clone())
    return torch.stack(O), torch.stack(ACT), torch.stack(R), torch.stack(D)


def _params(width, seed=4):
    g = torch.Generator(DEV).manual_seed(seed)
    shapes = [(width, 14), (width,), (width, width), (width,), (5, width), (5,), (1, width), (1,)]
    return [(torch.randn(s, device=DEV, generator=g) * (0.5 / math.sqrt(s[-1]) if len(s) == 2 else 0.1)) for s in shapes]


def _net(linear, p, x):
    h = linear(x, p[0], p[1], "tanh", None)
    h = linear(h, p[2], p[3], "gelu", h)
    return linear(h, p[4], p[5], None, None), linear(h, p[6], p[7], None, None).squeeze(-1)


def _linear64(x, w, b, act, r):
    z = x @ w.T + b
    y = torch.tanh(z) if act == "tanh" else z * 0.5 * torch.erfc(-z / math.sqrt(2)) if act == "gelu" else z
    return y if r is None else y + r


@pytest.mark.parametrize("width", [64, 37])
def test_policy_update_from_a_rollout(width):
    import mpe_hip
    lin = lambda x, w, b, act, r: mpe_hip.linear(x, w, b, activation=act, residual=r)
    O, ACT, R, D = _collect()
    old = _params(width)
    with torch.no_grad():
        logits0, values0 = _net(lin, old, O)
        lp0 = torch.log_softmax(logits0, -1).gather(-1, ACT.long()[..., None])[..., 0].contiguous()
    adv, ret = mpe_hip.gae(R, values0, D, values0[-1].contiguous())
    adv = (adv - adv.mean()) / (adv.std() + 1e-8)
    new = [(p + 0.02 * torch.randn(p.shape, device=DEV, generator=torch.Generator(DEV).manual_seed(9))).requires_grad_(True) for p in old]
    logits, values = _net(lin, new, O)
    loss, stats = mpe_hip.ppo_loss(logits, ACT, lp0, adv, values=values, old_values=values0, returns=ret, value_clip=None)
    loss.backward()
    # the same in float64, by autograd
    p64 = [p.detach().double().requires_grad_(True) for p in new]
    l64, v64 = _net(_linear64, p64, O.double())
    logp = torch.log_softmax(l64, -1)
    q = (logp.gather(-1, ACT.long()[..., None])[..., 0] - lp0.double()).exp()
    a64 = adv.double()
    # a row within 1e-5 of a clipping border may take either branch: the float64 side takes the kernel's, which float32 decides
    near = ((q.detach() - 0.8).abs() < 1e-5) | ((q.detach() - 1.2).abs() < 1e-5)
    assert not near.any()
    pg = -torch.minimum(q * a64, q.clamp(0.8, 1.2) * a64).mean()
    ent = -(logp.exp() * logp).sum(-1).mean()
    want = pg + 0.5 * 0.5 * ((v64 - ret.double()) ** 2).mean() - 0.01 * ent
    assert abs(float(loss) - float(want)) <= 1e-5 * (1 + abs(float(want)))
    g64 = torch.autograd.grad(want, p64)
    total = math.sqrt(sum(float((g ** 2).sum()) for g in g64))
    for p, g in zip(new, g64):      # float32 through three layers: 2^-24 per operation, a few hundred of them, of the whole gradient's size
        assert float((p.grad.double() - g).abs().max()) <= 2e-5 * total
    before = [p.grad.clone() for p in new]
    norm = mpe_hip.clip_grad_norm_(new, 0.5 * total)
    assert abs(float(norm) - total) <= 4e-5 * total
    for p, b in zip(new, before):
        assert torch.allclose(p.grad, b * (0.5 * total / norm), rtol=1e-6, atol=0)
    with torch.no_grad():
        for p in new:
            p -= 0.01 * p.grad
    l2, v2 = _net(lin, [p.detach() for p in new], O)
    assert torch.isfinite(l2).all() and torch.isfinite(v2).all() and stats.shape == (5,)


def test_whole_update_captured():
    """Layers, loss, gradients and clipping in one graph, replayed on new parameters."""
    import mpe_hip
    lin = lambda x, w, b, act, r: mpe_hip.linear(x, w, b, activation=act, residual=r)
    O, ACT, R, D = _collect(B=32, T=6)
    with torch.no_grad():
        l0, v0 = _net(lin, _params(48, 5), O)
        lp0 = torch.log_softmax(l0, -1).gather(-1, ACT.long()[..., None])[..., 0].contiguous()
    adv, ret = mpe_hip.gae(R, v0, D, v0[-1].contiguous())

    def update(ps):
        logits, values = _net(lin, ps, O)
        loss, stats = mpe_hip.ppo_loss(logits, ACT, lp0, adv, values=values, old_values=v0, returns=ret, value_clip=0.2)
        grads = torch.autograd.grad(loss, ps)
        clipped = [torch.empty_like(g) for g in grads]
        norm = mpe_hip.clip_grad_norm(grads, 0.1, out=clipped)
        return [loss.detach(), stats, norm] + clipped

    held = [p.clone().requires_grad_(True) for p in _params(48, 6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        update(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = update(held)
    for i in range(3):
        with torch.no_grad():
            for p, q in zip(held, _params(48, 20 + i)):
                p.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        want = update([p.detach().clone().requires_grad_(True) for p in held])
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        torch.cuda.synchronize()
