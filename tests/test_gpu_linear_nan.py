"""float32 layers whose data is not finite: the sums float32 has, at a cost that stays in proportion.

A result is summed again in plain float32 where the sum of its parts is not finite: off by (K + 8) 2^-24 of its sizes like any other."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
V = 2.0 ** -24
BIG = torch.finfo(torch.float32).max
# few rows in one and several column groups, small and large tiles, narrow, ragged
SHAPES = [(3, 14, 64), (16, 1024, 100), (40, 70, 90), (300, 33, 20), (2048, 64, 64), (5000, 17, 9), (3001, 258, 255), (9000, 130, 520), (20000, 64, 64), (70000, 14, 64)]


def make(m, k, n, seed=0):
    g = torch.Generator(DEV).manual_seed(seed + 7919 * m + 131 * k + n)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
    return rnd(m, k), rnd(n, k) / math.sqrt(k), rnd(n), rnd(m, n)


def same(got, a, b, bias=None):
    """got against a @ b.T (+ bias) in float64, whose infinities and NaN are float32's where nothing overflows."""
    want, mag = a.double() @ b.double().T, a.double().nan_to_num(0, 0, 0).abs() @ b.double().nan_to_num(0, 0, 0).abs().T
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    inf = want.isinf()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), inf) and torch.equal(got[inf].double(), want[inf])
    ok = want.isfinite()
    assert ((got.double() - want).abs() <= (a.shape[1] + 8) * V * mag + 2.0 ** -126)[ok].all()


def spoil(t, seed):
    """Infinities of both signs and NaN in a few places, none in most rows."""
    g = torch.Generator().manual_seed(seed)
    t = t.clone()
    for i in range(6):
        r, c = int(torch.randint(0, t.shape[0], (1,), generator=g)), int(torch.randint(0, t.shape[1], (1,), generator=g))
        t[r, c] = (math.inf, math.nan, -math.inf)[i % 3]
    t[t.shape[0] - 1, t.shape[1] - 1] = math.inf
    return t


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_forward_and_gradients_are_float32s(m, k, n):
    import mpe_hip
    x, w, b, dy = make(m, k, n)
    clean = mpe_hip.linear(x, w, b)
    for xx, ww in ((spoil(x, 1), w), (x, spoil(w, 2)), (spoil(x, 3), spoil(w, 4))):
        got = mpe_hip.linear(xx, ww, b)
        same(got, xx, ww, b)
        untouched = xx.isfinite().all(1)[:, None] & ww.isfinite().all(1)[None]
        assert torch.equal(got[untouched], clean[untouched])
        leaves = [xx.detach().requires_grad_(True), ww.detach().requires_grad_(True), b.detach().clone().requires_grad_(True)]
        y = mpe_hip.linear(*leaves)
        for up in (dy, spoil(dy, 5)):
            dx, dw, db = torch.autograd.grad(y, leaves, up, retain_graph=True)
            same(dx, up, ww.T)
            same(dw, up.T, xx.T)
            assert torch.equal(db.isnan(), up.double().sum(0).isnan())


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_numbers_that_round_to_infinity_in_their_first_part(m, k, n):
    """The top of float32's range is beyond bfloat16's: its first part is infinite and its products are made again."""
    import mpe_hip
    x, w, b, _ = make(m, k, n, seed=1)
    x[0, 0], x[m - 1, k - 1] = BIG, -BIG
    w[:, 0], w[:, k - 1] = w[:, 0].abs() * 2.0 ** -8, w[:, k - 1].abs() * 2.0 ** -8
    same(mpe_hip.linear(x, w, b), x, w, b)


def test_activations_and_residual_after_it():
    import mpe_hip
    x, w, b, r = make(300, 40, 72)
    x[7, 3], x[8, 4] = math.inf, math.nan
    w[:, 3] = w[:, 3].abs() + 0.1
    got = mpe_hip.linear(x, w, b, "tanh", r)
    assert torch.equal(got[7], 1 + r[7]) and got[8].isnan().all() and got[:7].isfinite().all() and got[9:].isfinite().all()


@pytest.mark.parametrize("m,k,n,times", [(16384, 1024, 1024, 10), (4, 1024, 1024, 8), (65536, 64, 64, 10)])
def test_the_time_stays_in_proportion(m, k, n, times):
    """Plain float32 sums run at about a quarter of the rate of those on the matrix cores, by the instructions, and both are made."""
    import mpe_hip
    x, w, b, _ = make(m, k, n)
    def best(x, w):
        mpe_hip.linear(x, w, b)
        out = []
        for _ in range(5):
            one, two = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            one.record()
            for _ in range(10):
                mpe_hip.linear(x, w, b)
            two.record()
            two.synchronize()
            out.append(one.elapsed_time(two))
        return min(out)
    finite = best(x, w)
    w2 = w.clone()
    w2[5] = math.nan
    row, everything = best(x, w2), best(torch.full_like(x, math.nan), w)
    print("\n%d x %d -> %d: %.1f us, a NaN row of weights %.1f, all NaN %.1f" % (m, k, n, finite * 100, row * 100, everything * 100))
    assert row <= times * finite and everything <= times * finite


@pytest.mark.parametrize("power", [-60, -100, -109, -112, -116, -120])
def test_numbers_far_down_in_float32(power):
    """The parts of a number end with bfloat16's smallest, 2^-133: below 2^-109 what lies under half of it, 2^-134, is lost of every
    factor, and nothing else."""
    import mpe_hip
    for m, k, n in ((5, 40, 30), (300, 100, 72), (5000, 17, 200)):
        x, w, b, dy = make(m, k, n, seed=2)
        for xx, ww, other in ((x * 2.0 ** power, w, w.double().abs().sum(1)[None]), (x, w * 2.0 ** power, x.double().abs().sum(1)[:, None])):
            lost = 2.0 ** -134 * other
            got, want = mpe_hip.linear(xx, ww), xx.double() @ ww.double().T
            mag = xx.double().abs() @ ww.double().abs().T
            assert ((got.double() - want).abs() <= (k + 8) * V * mag + lost + 2.0 ** -149).all()
