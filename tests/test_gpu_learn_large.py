"""mpe_hip.linear, ppo_loss and clip_grad_norm on tensors of more than 2^31 elements, and under inference mode.  What is looked
at are the first and last rows, which an offset of 32 bits would miss; bounds as in test_gpu_linear.py: (K + 8) 2^-24 of the
sum of the products' sizes, one rounding of 2^-8, and where dz is rounded first 2^-8 of those sizes more."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
V, U = 2.0 ** -24, 2.0 ** -8


def inside(got, want, bound):
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), float((d / bound).max())


def rand(*shape, seed):
    return torch.randn(*shape, device=DEV, dtype=torch.bfloat16, generator=torch.Generator(DEV).manual_seed(seed))


def test_linear_with_more_than_2_to_31_weights():
    import mpe_hip
    m, k, n = 24, 40960, 54000
    x, w = rand(m, k, seed=1).requires_grad_(True), rand(n, k, seed=2).requires_grad_(True)
    y = mpe_hip.linear(x, w, activation="relu")
    dy = rand(m, n, seed=3)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    rows = torch.tensor([0, 1, 26213, 26214, 52428, 52429, n - 2, n - 1], device=DEV)
    xd, wd = x.detach().double(), w.detach()[rows].double()
    z = xd @ wd.T
    size = xd.abs() @ wd.abs().T
    inside(y[:, rows], z.clamp(min=0), (k + 8) * V * size + U * z.abs())
    dz = torch.where(y.detach()[:, rows] > 0, dy[:, rows], torch.zeros((), device=DEV, dtype=dy.dtype)).double()
    inside(dw[rows], dz.T @ xd, (m + 8) * V * (dz.abs().T @ xd.abs()) + U * (dz.T @ xd).abs())
    cols = torch.tensor([0, k - 1], device=DEV)
    dzf = torch.where(y.detach() > 0, dy, torch.zeros((), device=DEV, dtype=dy.dtype)).double()
    wc = w.detach()[:, cols].double()
    inside(dx[:, cols], dzf @ wc, (n + 8) * V * (dzf.abs() @ wc.abs()) + U * (dzf @ wc).abs())


def test_linear_with_more_than_2_to_31_inputs():
    import mpe_hip
    m, k, n = 34_000_001, 64, 64
    x = rand(m, k, seed=4).requires_grad_(True)
    w, b = rand(n, k, seed=5).requires_grad_(True), rand(n, seed=6).requires_grad_(True)
    y = mpe_hip.linear(x, w, b)
    rows = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, (1 << 25) + 1, m - 2, m - 1], device=DEV)
    xd, wd = x.detach()[rows].double(), w.detach().double()
    z = xd @ wd.T + b.detach().double()
    inside(y[rows], z, (k + 9) * V * (xd.abs() @ wd.abs().T + b.detach().double().abs()) + U * z.abs())
    dy = torch.zeros_like(y)
    dy[rows] = rand(len(rows), n, seed=7)       # the others add zeros: exact
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    d = dy[rows].double()
    inside(dx[rows], d @ wd, (n + 8) * V * (d.abs() @ wd.abs()) + U * (d @ wd).abs())
    inside(dw, d.T @ xd, (len(rows) + 8) * V * (d.abs().T @ xd.abs()) + U * (d.T @ xd).abs())
    inside(db, d.sum(0), (len(rows) + 8) * V * d.abs().sum(0) + U * d.sum(0).abs())


def test_ppo_loss_with_more_than_2_to_31_logits():
    """Only the first and the last rows have weight, so a few rows alone must give the same loss and gradients."""
    import mpe_hip
    rows, v = 270_001, 8000
    logits = rand(rows, v, seed=8).requires_grad_(True)
    g = torch.Generator(DEV).manual_seed(9)
    actions = torch.randint(0, v, (rows,), device=DEV, generator=g)
    old, adv = -9 + torch.randn(rows, device=DEV, generator=g), torch.randn(rows, device=DEV, generator=g)
    some = torch.tensor([0, 1, 268_434, 268_435, 268_436, rows - 2, rows - 1], device=DEV)
    weights = torch.zeros(rows, device=DEV)
    weights[some] = 1.0
    loss, stats = mpe_hip.ppo_loss(logits, actions, old, adv, weights=weights)
    grad, = torch.autograd.grad(loss, logits)
    few = logits.detach()[some].clone().requires_grad_(True)
    want, wstats = mpe_hip.ppo_loss(few, actions[some], old[some], adv[some])
    wgrad, = torch.autograd.grad(want, few)
    # the same float64 sums of the same seven numbers in another order, rounded to float32 once
    assert torch.allclose(loss, want, rtol=2.0 ** -22, atol=0) and torch.allclose(stats, wstats, rtol=2.0 ** -22, atol=0)
    assert torch.equal(grad[some], wgrad)
    grad[some] = 0
    assert not grad.any()


def test_clip_of_more_than_2_to_31_elements():
    import mpe_hip
    big = torch.zeros((1 << 31) + 77, device=DEV, dtype=torch.bfloat16)
    big[0], big[1 << 31], big[-1] = 1.0, 2.0, 2.0
    norm = mpe_hip.clip_grad_norm([big], 1.5, out=[big])
    assert float(norm) == 3.0 and [float(big[i]) for i in (0, 1 << 31, -1)] == [0.5, 1.0, 1.0]
    assert float(mpe_hip.grad_norm([big])) == 1.5


def test_clip_of_a_thousand_tensors():
    import mpe_hip
    ts = [torch.full((37 + i % 5000,), 0.25, device=DEV, dtype=(torch.float32, torch.bfloat16, torch.float16)[i % 3]) for i in range(1000)]
    total = sum(t.numel() for t in ts)
    norm = mpe_hip.clip_grad_norm(ts, 1.0, out=ts)
    want = 0.25 * total ** 0.5
    assert abs(float(norm) - want) <= 2 * V * want
    for t in ts:        # two float32 roundings (the factor, the product), then the type's
        off = (2 * V + torch.finfo(t.dtype).eps / 2) * 0.25 / want
        assert float((t.double() - 0.25 / want).abs().max()) <= 1.01 * off, t.dtype


def test_under_inference_mode():
    import mpe_hip
    x, w = rand(70, 40, seed=10), rand(24, 40, seed=11)
    logits, a = torch.randn(70, 5, device=DEV), torch.zeros(70, dtype=torch.int32, device=DEV)
    z = torch.zeros(70, device=DEV)
    want, (loss, stats) = mpe_hip.linear(x, w, activation="gelu"), mpe_hip.ppo_loss(logits, a, z, z + 1)
    with torch.inference_mode():
        assert torch.equal(mpe_hip.linear(x, w, activation="gelu"), want)
        l2, s2 = mpe_hip.ppo_loss(logits, a, z, z + 1)
        assert torch.equal(l2, loss) and torch.equal(s2, stats)
        g = torch.ones(9, device=DEV)
        assert float(mpe_hip.clip_grad_norm([g], 1.5, out=[g])) == 3.0 and torch.equal(g, torch.full_like(g, 0.5))
