"""Layers of which some parts are frozen: a gradient's bits do not depend on which others are asked for, and one that is not asked
for costs nothing."""
import itertools

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1, 1), (2, 3, 2), (1, 100, 1), (33, 10, 7), (1000, 14, 64), (5000, 64, 64), (3001, 258, 255), (700, 70, 90), (40000, 33, 20), (8200, 320, 1032), (5000, 260, 300), (70001, 66, 3)]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu", "tanh", "gelu"])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_every_subset_gives_the_same_bits(m, k, n, act, dt):
    import mpe_hip
    g = torch.Generator(DEV).manual_seed(m + k + n)
    x, w, b, dy = [torch.randn(*s, device=DEV, generator=g).to(dt) for s in ((m, k), (n, k), (n,), (m, n))]
    full = None
    for need in itertools.product((True, False), repeat=3):
        if not any(need):
            continue
        leaves = [t.detach().clone().requires_grad_(q) for t, q in zip((x, w, b), need)]
        y = mpe_hip.linear(*leaves, act)
        got = iter(torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy))
        got = [next(got) if q else None for q in need]
        full = full or got
        assert all(q is None or torch.equal(q, f) for q, f in zip(got, full)), need


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("m,k,n", [(40, 6, 9), (1000, 14, 64), (3001, 258, 255), (8200, 320, 1032)])
def test_subsets_with_upstream_gradients_that_are_not_rows(m, k, n, act, dt):
    """One row for all, columns of a wider tensor, a transposed one: the same bits from every subset (their alignment may choose another
    kernel than a contiguous tensor's)."""
    import mpe_hip
    g = torch.Generator(DEV).manual_seed(m + k + n)
    x, w, b, wide = [torch.randn(*s, device=DEV, generator=g).to(dt) for s in ((m, k), (n, k), (n,), (m, n + 3))]
    for dy in (wide[:1, :n].expand(m, n), wide[:, 1:n + 1], wide[:, :n].T.contiguous().T):
        def grads(need, up):
            leaves = [t.detach().clone().requires_grad_(q) for t, q in zip((x, w, b), need)]
            got = iter(torch.autograd.grad(mpe_hip.linear(*leaves, act), [t for t in leaves if t.requires_grad], up))
            return [next(got) if q else None for q in need]
        want = grads((True, True, True), dy)
        for need in ((False, False, True), (True, False, True), (False, True, False), (True, False, False)):
            assert all(q is None or torch.equal(q, f) for q, f in zip(grads(need, dy), want)), need


@pytest.mark.parametrize("m,k,n,act,dt", [(65536, 1024, 1024, "none", torch.float32), (65536, 1024, 1024, "none", torch.bfloat16), (65536, 512, 512, "gelu", torch.float32),
                                          (65536, 512, 500, "gelu", torch.float16)])
def test_a_bias_alone_costs_no_product(m, k, n, act, dt):
    """Column sums read dy and what was kept once; the weights' product beside them takes several times as long at these sizes."""
    import mpe_hip
    x, w, b, dy = [torch.randn(*s, device=DEV).to(dt) for s in ((m, k), (n, k), (n,), (m, n))]
    def best(leaves):
        y = mpe_hip.linear(x, w, b, act)
        out = []
        for _ in range(6):
            one, two = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            one.record()
            for _ in range(5):
                torch.autograd.grad(y, leaves, dy, retain_graph=True)
            two.record()
            two.synchronize()
            out.append(one.elapsed_time(two) * 200)
        return min(out)
    b.requires_grad_(True)
    alone = best([b])
    w.requires_grad_(True)
    both = best([w, b])
    print("\n%d x %d -> %d %s: bias %.1f us, with the weights %.1f" % (m, k, n, act, alone, both))
    assert alone <= 0.6 * both
