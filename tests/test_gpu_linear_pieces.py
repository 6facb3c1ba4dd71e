"""The gradients of mpe_hip.linear in 16-bit types: dz enters the products with twice the type's bits and a gradient is rounded
once.

Bounds, written down before any run, with u half a step of the type (bf16 2^-8, fp16 2^-11) and v = 2^-24: a sum of K terms is off
by (K + 8) v of their sizes, a pre-activation by (k + 8) v of its, a slope by at most 0.9 of that, 16 v (1 + |z|) of its own and, in
bfloat16, which keeps slopes in float16, by 2^-11 of itself; dz in two pieces is off by u^2 |dz| and, in float16, by half a step of
its smallest number over 2^10 (the rests are kept 2^11 times as large, of half of dz); then one rounding, u of the result."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
V = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
HALVES = [torch.bfloat16, torch.float16]


def act64(z, act):
    return {"none": lambda: z, "tanh": lambda: torch.tanh(z), "gelu": lambda: z * 0.5 * torch.erfc(-z / math.sqrt(2)), "silu": lambda: z * torch.sigmoid(z)}[act]()


def slope64(z, act):
    z = z.detach().requires_grad_(True)
    with torch.enable_grad():
        return torch.autograd.grad(act64(z, act).sum(), z)[0]


def gradients(x, w, b, dy, act):
    """The kernels' dx, dw, db, and float64's with the sizes of what they sum and of what dz may be off by."""
    import mpe_hip
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(mpe_hip.linear(*leaves, act), leaves, dy)
    xd, wd, dt, k = x.double(), w.double(), x.dtype, x.shape[1]
    z = xd @ wd.T + b.double()
    size = xd.abs() @ wd.abs().T + b.double().abs()
    d = dy.double()
    dz = d * slope64(z, act)
    e = U[dt] ** 2 * dz.abs() + TINY[dt] * 2.0 ** -10
    if act != "none":
        e = e + d.abs() * (0.9 * (k + 8) * V * size + 16 * V * (1 + z.abs())) + (2.0 ** -11 if dt == torch.bfloat16 else 0.0) * dz.abs()
    return got, dz, e


def check(x, w, b, dy, act):
    (dx, dw, db), dz, e = gradients(x, w, b, dy, act)
    dt, (m, n) = x.dtype, dz.shape
    xd, wd = x.double(), w.double()
    for name, got, want, mag, off in (("dx", dx, dz @ wd, dz.abs() @ wd.abs(), (n + 8, e @ wd.abs())), ("dw", dw, dz.T @ xd, dz.abs().T @ xd.abs(), (m + 8, e.T @ xd.abs())),
                                      ("db", db, dz.sum(0), dz.abs().sum(0), (m + 8, e.sum(0)))):
        bound = off[0] * V * (mag + off[1]) + off[1]
        bound = bound * (1 + U[dt]) + U[dt] * want.abs() + TINY[dt]
        bad = ~((got.double() - want).abs() <= bound)
        if dt == torch.float16:         # 65520 is where rounding to float16 becomes infinite: an infinity is right from there on
            bad &= ~((got.double() == torch.copysign(torch.full_like(want, math.inf), want)) & (want.abs() + bound >= 65520.0))
        assert not bad.any(), "%s: %d of %d outside, worst %g" % (name, int(bad.sum()), bad.numel(), float(((got.double() - want).abs() / bound).max()))


def make(m, k, n, dt, ld=None, seed=0):
    g = torch.Generator(DEV).manual_seed(seed + 7919 * m + 131 * k + n)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
    ld = ld or k
    return rnd(m, ld).to(dt)[:, ld - k:], (rnd(n, k) / math.sqrt(k)).to(dt), rnd(n).to(dt), rnd(m, n).to(dt)


# copies to LDS, whole and ragged; an odd row stride and odd widths that keep them out, in large and small tiles; narrow inputs
SHAPES = [(8192, 256, 1024, 256), (8200, 320, 1032, 320), (16421, 264, 520, 264), (5000, 1000, 1304, 1001), (5000, 1001, 300, 1001), (3001, 258, 255, 258), (700, 70, 90, 70),
          (3000, 64, 64, 64), (2000, 14, 64, 42), (900, 40, 17, 40), (300, 9, 130, 9)]


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n,ld", SHAPES)
def test_the_error_is_one_rounding(m, k, n, ld, dt):
    """Root mean square against that of float64's gradients rounded once.  What bfloat16's slopes add is an eighth of a rounding,
    1 + 1/128; the sums' float32 far less."""
    x, w, b, dy = make(m, k, n, dt, ld)
    (dx, dw, _), dz, _ = gradients(x, w, b, dy, "gelu")
    for got, want in ((dx, dz @ w.double()), (dw, dz.T @ x.double())):
        least = float((want.to(dt).double() - want).norm())
        assert float((got.double() - want).norm()) <= 1.02 * least + 1e-12


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("act", ["gelu", "tanh", "silu", "none"])
@pytest.mark.parametrize("m,k,n,ld", SHAPES)
def test_sums_of_one_term_and_sums_that_cancel(m, k, n, ld, act, dt):
    """Weights with one or two (opposite) entries a column and inputs with one or two a column: a rounding of dz has nothing to hide
    behind."""
    x, w, b, dy = make(m, k, n, dt, ld, seed=1)
    col = torch.arange(k, device=DEV)
    few = torch.zeros_like(w)
    few[col % n, col] = w[col % n, col] + 0.75
    check(x, few, b, dy, act)
    few[(col + 1) % n, col] = -few[col % n, col]
    near = dy.clone()
    near[:, 1:] = dy[:, :1]
    check(x, few, torch.zeros_like(b) if n > 1 else b, near, act)
    rows = torch.zeros_like(x)
    at = (col * 37) % m
    rows[at, col] = x[at, col] + 0.75
    check(rows, w, b, dy, act)
    rows[(at + 1) % m, col] = -rows[at, col]
    check(rows, w, b, dy[:1].expand(m, n) if act == "none" else dy[:1].expand(m, n).contiguous(), act)


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n,ld", SHAPES)
def test_dense_sums(m, k, n, ld, dt):
    check(*make(m, k, n, dt, ld, seed=2), "gelu")


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n,ld", SHAPES)
def test_infinities_and_nan_reach_what_they_would(m, k, n, ld, dt):
    """Where float32's sums are infinite or NaN the gradients are, and nowhere else; dz stays clear of zero."""
    import mpe_hip
    x, w, b, dy = make(m, k, n, dt, ld, seed=3)
    b = b.abs() + 1
    x, w = x * 0.25, w * 0.25
    dy = (dy.abs() + 0.5) * torch.where(dy < 0, -1, 1)
    z = torch.nn.functional.linear(x.float(), w.float(), b.float())
    dz = dy.float() * slope64(z, "silu").float()
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    y = mpe_hip.linear(*leaves, "silu")
    bad = dy.clone()
    bad[3, 0], bad[5, n // 2], bad[m - 1, n - 1] = math.inf, math.nan, -math.inf
    dz = torch.where(torch.isfinite(bad.float()), dz, bad.float())
    got = torch.autograd.grad(y, leaves, bad)
    for a, want in zip(got, (dz @ w.float(), dz.T @ x.float(), dz.sum(0))):
        assert torch.equal(a.isnan(), want.isnan())
        assert torch.equal(a.isinf(), want.isinf()) and torch.equal(a[a.isinf()].float(), want[want.isinf()])
    # the same in the other operand of each product: the forward pass has to be finite, so the leaves change under it
    dz = dy.float() * slope64(z, "silu").float()
    for name in ("w", "x"):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
        y = mpe_hip.linear(*leaves, "silu")
        t = leaves[1 if name == "w" else 0].data
        t[2, 1], t[t.shape[0] - 1, k - 1] = math.inf, math.nan
        got = torch.autograd.grad(y, leaves, dy)
        a, want = (got[0], dz @ t.float()) if name == "w" else (got[1], dz.T @ t.float())
        assert torch.equal(a.isnan(), want.isnan()), name
        assert torch.equal(a.isinf(), want.isinf()) and torch.equal(a[a.isinf()].float(), want[want.isinf()]), name


@pytest.mark.parametrize("m,k,n,ld", SHAPES)
@pytest.mark.parametrize("power", [-20, -16, -12, -8])
def test_float16_gradients_keep_their_bits_where_dz_is_small(m, k, n, ld, power):
    """dy far down in float16's range: its own few bits are all that is lost.  The other operands are as much larger, so that the
    results lie where float16 has all its bits; x and w in turn, so that pre-activations stay where slopes are between 0 and 1."""
    x, w, b, dy = make(m, k, n, torch.float16, ld, seed=4)
    dy = dy * 2.0 ** power
    up = 2.0 ** min(-power - 6, 9)
    check(x * up, w / up, b, dy, "silu")
    check(x / up, w * up, b, dy, "silu")


@pytest.mark.parametrize("m,k,n,ld", SHAPES)
def test_float16_gradients_are_finite_where_dz_is_beyond_its_range(m, k, n, ld):
    """gelu's slope is 1.13 at 1.41: dy of 60000 gives dz of 67000."""
    x, w, b, dy = make(m, k, n, torch.float16, ld, seed=5)
    x, w, b = x * 2.0 ** -8, w * 2.0 ** -6, torch.full_like(b, 1.41)
    dy = torch.where(dy < 0, -60000.0, 60000.0).half()
    got, dz, _ = gradients(x, w, b, dy, "gelu")
    assert float(dz.abs().max()) > 65504 * 1.02
    check(x, w, b, dy, "gelu")


@pytest.mark.parametrize("m,k,n", [(513, 1, 1), (513, 14, 20), (513, 70, 40), (8192, 64, 1024), (8193, 264, 520)])
@pytest.mark.parametrize("act", ["tanh", "silu"])
def test_bfloat16_keeps_small_slopes_to_their_own_precision(m, k, n, act):
    """Saturated units: slopes down to 2^-28, where 2^14 times them leave float16's normal range.  One term in every sum.  Off by the
    kept slope's rounding 2^-11, by the exponential's (2 |z| + 8) 2^-22 and, silu's only, by 2^-22 of the size of its two terms, and
    rounded once."""
    import mpe_hip
    dt = torch.bfloat16
    z = torch.linspace(-9.5, 9.5, m, device=DEV).to(dt)
    x, w, dy = torch.zeros(m, k, device=DEV, dtype=dt), torch.zeros(n, k, device=DEV, dtype=dt), torch.zeros(m, n, device=DEV, dtype=dt)
    x[:, 0], w[n - 1, 0], dy[:, n - 1] = z, 1.0, 3.0
    x.requires_grad_(True)
    got, = torch.autograd.grad(mpe_hip.linear(x, w, None, act), x, dy)
    zd = z.double()
    slope = 1 / torch.cosh(zd) ** 2 if act == "tanh" else torch.sigmoid(zd) * (1 + zd * torch.sigmoid(-zd))
    parts = slope if act == "tanh" else torch.sigmoid(zd) * (1 + zd.abs())
    off = 3 * (slope.abs() * 2.0 ** -11 + parts * (2 * zd.abs() + 8) * 2.0 ** -22 + 2.0 ** -39)
    assert ((got[:, 0].double() - 3 * slope).abs() <= off + U[dt] * (3 * slope.abs() + off)).all()
    assert float(got[:, 1:].abs().sum()) == 0


@pytest.mark.parametrize("m,k,n", [(4_200_001, 256, 520), (4_200_001, 259, 513)])
def test_pieces_of_more_than_2_to_32_elements(m, k, n):
    """Both pieces of dz together; first, middle and last rows, which an offset of 32 bits would miss."""
    import mpe_hip
    dt = torch.bfloat16
    rnd = lambda *s, seed: torch.randn(*s, device=DEV, dtype=dt, generator=torch.Generator(DEV).manual_seed(seed))
    x, w = rnd(m, k, seed=1).requires_grad_(True), (rnd(n, k, seed=2) / 16).requires_grad_(True)
    y = mpe_hip.linear(x, w, None, "silu")
    rows = torch.tensor([0, 1, 2 ** 31 // n - 1, 2 ** 31 // n, 2 ** 31 // n + 1, 2 ** 32 // (2 * n), 2 ** 32 // n // 2 + 1, m - 2, m - 1], device=DEV).unique()
    dy = torch.zeros_like(y)
    dy[rows] = rnd(len(rows), n, seed=3)            # the others add zeros: exact
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    xd, wd, d = x.detach()[rows].double(), w.detach().double(), dy[rows].double()
    z = xd @ wd.T
    dz = d * slope64(z, "silu")
    e = d.abs() * (0.9 * (k + 8) * V * (xd.abs() @ wd.abs().T) + 16 * V * (1 + z.abs())) + (2.0 ** -11 + U[dt] ** 2) * dz.abs()
    for got, want, off, mag, terms in ((dx[rows], dz @ wd, e @ wd.abs(), dz.abs() @ wd.abs(), n), (dw, dz.T @ xd, e.T @ xd.abs(), dz.abs().T @ xd.abs(), len(rows))):
        bound = off + (terms + 8) * V * (mag + off)
        assert ((got.double() - want).abs() <= bound * (1 + U[dt]) + U[dt] * want.abs() + TINY[dt]).all()
    other = torch.ones(m, dtype=torch.bool, device=DEV)
    other[rows] = False
    assert float(dx[other].abs().max()) == 0


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n", [(16384, 256, 512), (3001, 258, 255), (3000, 64, 64)])
def test_captured_gradients_replay(m, k, n, dt):
    """A captured forward and backward pass beside a second one of the same leaves, replayed between eager calls on new inputs."""
    import mpe_hip
    x, w, b, dy = make(m, k, n, dt)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    call = lambda ls, up: torch.autograd.grad(mpe_hip.linear(*ls, "gelu"), ls, up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(leaves, dy)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(call(leaves, dy))
    for i in range(3):
        with torch.no_grad():
            for t in leaves:
                t.copy_(torch.randn_like(t) * 0.3)
            dy.copy_(torch.randn_like(dy))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = call([t.detach().clone().requires_grad_(True) for t in leaves], dy)
        for out in outs:
            assert all(torch.equal(p, q) for p, q in zip(out, want)), i
        torch.cuda.synchronize()


@pytest.mark.parametrize("dt", HALVES)
@pytest.mark.parametrize("m,k,n,ld", SHAPES)
def test_relus_dz_is_exact_in_one_piece(m, k, n, ld, dt):
    """dy or zero: sums of one term are products rounded once, and dense ones are off by no more than their float32 order."""
    import mpe_hip
    x, w, b, dy = make(m, k, n, dt, ld, seed=6)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    y = mpe_hip.linear(*leaves, "relu")
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    dz = torch.where(y.detach() > 0, dy, torch.zeros_like(dy)).double()
    xd, wd = x.double(), w.double()
    for got, want, mag, terms in ((dx, dz @ wd, dz.abs() @ wd.abs(), n), (dw, dz.T @ xd, dz.abs().T @ xd.abs(), m), (db, dz.sum(0), dz.abs().sum(0), m)):
        off = (terms + 8) * V * mag
        assert ((got.double() - want).abs() <= off + U[dt] * (want.abs() + off) + TINY[dt]).all()
