"""mpe_hip.linear against the formula in float64, element by element.

The bounds are the arithmetic's worst case, written down before any run.  u = half a step of the type (bf16 2^-8, fp16 2^-11,
fp32 2^-24), v = 2^-24.  A sum of K products in 32 bits is off by at most (K + 8) v sum |x||w| whatever its order (a float32
product that is summed from parts in 16 bits included: what the parts drop stays below 4 v |x||w|), an activation of slope at
most 1.13 carries that on and adds a few v of its own value, and the result is rounded once: u |y|.  The backward pass reads
pre-activations rounded to the type at worst (u |z|, and the slopes change by at most 0.9 a unit of z), rounds dz once (u |dz|)
and sums like the forward; smallest numbers add one underflow step.  bfloat16 keeps the slopes themselves in float16, which is
2^-11 |dz| more where z is small and the bound by u |z| does not cover it."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
V = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
ACTS = ["none", "tanh", "relu", "gelu", "silu"]


def act64(z, act):
    return {"none": lambda: z, "tanh": lambda: torch.tanh(z), "relu": lambda: torch.clamp(z, min=0),
            "gelu": lambda: z * 0.5 * torch.erfc(-z / math.sqrt(2)), "silu": lambda: z * torch.sigmoid(z)}[act]()


def slope64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "tanh":
        return 1 - torch.tanh(z) ** 2
    if act == "relu":
        return (z > 0).double()
    if act == "gelu":
        return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def make(m, k, n, dt, seed=0, bias=True, residual=False, ld=None, exact=False):
    """exact: multiples of 1/4 up to 1, whose sums are exact in every type here, so that relu's border is the same everywhere."""
    g = torch.Generator(DEV).manual_seed(seed + 7919 * m + 131 * k + n)
    rnd = (lambda *s: torch.randint(-4, 5, s, device=DEV, generator=g).float() / 4) if exact else (lambda *s: torch.randn(*s, device=DEV, generator=g))
    ld = ld or k
    x = rnd(m, ld).to(dt)[:, ld - k:]
    w = (rnd(n, k) if exact else rnd(n, k) / math.sqrt(k)).to(dt)
    return x, w, (rnd(n).to(dt) if bias else None), (rnd(m, n).to(dt) if residual else None), rnd(m, n).to(dt)


def forward64(x, w, b, r, act):
    x, w = x.double(), w.double()
    z = x @ w.T
    size = x.abs() @ w.abs().T
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    y = act64(z, act)
    return z, size, (y if r is None else y + r.double())


def forward_bound(z, size, y, r, act, k, dt):
    off = (k + 8) * V * size * (1.13 if act in ("gelu", "silu") else 1.0) + 8 * V * (act64(z, act).abs() + z.abs() * (act != "none"))
    if r is not None:
        off = off + 2 * V * (r.double().abs() + y.abs())
    return off + U[dt] * (y.abs() + off) + TINY[dt]


def inside(got, want, bound, what):
    d = (got.double() - want).abs()
    bad = ~(d <= bound)
    assert not bad.any(), "%s: %d of %d outside, worst off by %g times the bound" % (what, int(bad.sum()), bad.numel(), float((d / bound).max()))


def check_forward(x, w, b, r, act):
    import mpe_hip
    got = mpe_hip.linear(x, w, b, activation=act, residual=r)
    z, size, y = forward64(x, w, b, r, act)
    assert got.dtype == x.dtype and got.shape == x.shape[:-1] + (w.shape[0],)
    inside(got, y, forward_bound(z, size, y, r, act, x.shape[-1], x.dtype), "y")


def check_backward(x, w, b, r, dy, act, need_x=True):
    import mpe_hip
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    xx, ww = next(it), next(it)
    bb = next(it) if b is not None else None
    rr = next(it) if r is not None else None
    if not need_x:
        xx = x.detach()
    y = mpe_hip.linear(xx, ww, bb, activation=act, residual=rr)
    grads = torch.autograd.grad(y, leaves if need_x else leaves[1:], dy)
    dt = x.dtype
    m, k, n = x.shape[0], x.shape[1], w.shape[0]
    z, size, _ = forward64(x, w, b, r, act)
    sl, d = slope64(z, act), dy.double()
    dz = d * sl
    zoff = 0.0 if act in ("none", "relu") else 0.9 * (U[dt] * z.abs() + (k + 8) * V * size)
    e = d.abs() * (zoff + 16 * V * (1 + z.abs())) * (act != "none") + (U[dt] + (2.0 ** -11 if dt == torch.bfloat16 else 0)) * dz.abs() * (1 + U[dt]) + TINY[dt]
    xd, wd = x.double(), w.double()
    it = iter(grads)
    if need_x:
        want, mag = dz @ wd, dz.abs() @ wd.abs()
        off = e @ wd.abs() + (n + 8) * V * (mag + e @ wd.abs())
        inside(next(it), want, off * (1 + U[dt]) + U[dt] * want.abs() + TINY[dt], "dx")
    want, mag = dz.T @ xd, dz.abs().T @ xd.abs()
    off = e.T @ xd.abs() + (m + 8) * V * (mag + e.T @ xd.abs())
    inside(next(it), want, off * (1 + U[dt]) + U[dt] * want.abs() + TINY[dt], "dw")
    if b is not None:
        want, mag = dz.sum(0), dz.abs().sum(0)
        off = e.sum(0) + (m + 8) * V * (mag + e.sum(0))
        inside(next(it), want, off * (1 + U[dt]) + U[dt] * want.abs() + TINY[dt], "db")
    if r is not None:
        assert torch.equal(next(it), dy)


SHAPES = [(1, 1, 1), (1, 14, 64), (3, 14, 64), (4, 1024, 512), (16, 33, 5), (17, 31, 65), (63, 258, 33), (64, 64, 64), (65, 127, 129), (130, 3, 1), (200, 70, 5),
          (257, 96, 130), (513, 520, 250), (1000, 14, 64), (2000, 8, 300), (129, 4000, 17), (4099, 66, 63)]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_forward(m, k, n, dt):
    i = SHAPES.index((m, k, n))
    x, w, b, r, _ = make(m, k, n, dt, bias=i % 3 != 1, residual=i % 2 == 1)
    check_forward(x, w, b, r, ["tanh", "gelu", "silu", "none"][i % 4])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_every_activation_both_ways(act, dt):
    for m, k, n in ((70, 40, 72), (5, 12, 9)):
        x, w, b, r, dy = make(m, k, n, dt, residual=True, exact=act == "relu")
        check_forward(x, w, b, r, act)
        check_backward(x, w, b, r, dy, act)
        check_backward(x, w, b, None, dy, act)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_backward(m, k, n, dt):
    i = SHAPES.index((m, k, n))
    x, w, b, r, dy = make(m, k, n, dt, bias=i % 3 != 1, residual=i % 4 == 1)
    check_backward(x, w, b, r, dy, ["gelu", "tanh", "none", "silu"][i % 4], need_x=i % 5 != 4)


@pytest.mark.parametrize("dt", DTYPES)
def test_the_smallest_matrices(dt):
    """Operands shorter than a vector, and matrices that end inside one, in every combination."""
    for m in (1, 2, 3, 7, 9):
        for k in (1, 2, 3, 5, 7, 8, 9, 15):
            for n in (1, 2, 3, 4, 6, 7, 9):
                x, w, b, r, dy = make(m, k, n, dt, residual=(m + k + n) % 2 == 0)
                check_forward(x, w, b, r, "tanh")
                check_backward(x, w, b, r, dy, "tanh")
    for k, ld in ((1, 3), (3, 4), (5, 7)):
        x, w, b, r, dy = make(70, k, 3, dt, ld=ld)
        check_forward(x, w, b, r, "silu")
        check_backward(x, w, b, r, dy, "silu")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n", [1, 5, 12, 130])
def test_matrices_that_end_where_memory_ends(dt, n):
    """The last row's last vector: inputs that are the last elements of their buffers, with NaN all around them, give the same
    as inputs that stand alone."""
    import mpe_hip
    for m, k in ((65, 33), (129, 14), (40, 258), (300, 7)):
        x, w, b, r, dy = make(m, k, n, dt, residual=True)
        def framed(t):
            flat = torch.full((t.numel() + 64,), math.nan, device=DEV).to(dt)
            v = flat[33:33 + t.numel()].view(t.shape)
            v.copy_(t)
            return v
        for act in ("gelu", "relu", "none"):
            a = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
            f = [framed(t).requires_grad_(True) for t in (x, w, b, r)]
            one, two = (mpe_hip.linear(q[0], q[1], q[2], activation=act, residual=q[3]) for q in (a, f))
            assert torch.equal(one, two)
            assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(one, a, dy), torch.autograd.grad(two, f, framed(dy))))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n,ld", [(8192, 256, 1024, 256), (8200, 320, 1032, 320), (16421, 258, 512, 258), (70001, 72, 136, 74), (4097, 512, 264, 514),
                                      (5000, 1000, 1304, 1001)])
def test_large_products(m, k, n, ld, dt):
    """The sizes that take the copies to LDS, whole and ragged in every direction, and one whose odd row stride keeps them out."""
    x, w, b, r, dy = make(m, k, n, dt, residual=True, ld=ld)
    check_forward(x, w, b, r, "gelu")
    check_backward(x, w, b, r, dy, "silu")
    check_backward(x, w, b, None, dy, "none")


@pytest.mark.parametrize("m,k,n", [(1884, 817, 1), (8192, 256, 128), (5000, 70, 37), (3001, 1000, 300)])
def test_bias_gradient_sums_what_is_not_rounded(m, k, n):
    """Its terms cancel: float16 dz rounded before the sum would be off by up to 2^-11 of their sizes; the float32 sum and the
    slopes of float32 pre-activations are off by the arithmetic's bound without that."""
    import mpe_hip
    dt = torch.float16
    x, w, b, _, dy = make(m, k, n, dt)
    b.requires_grad_(True)
    db, = torch.autograd.grad(mpe_hip.linear(x, w, b, "tanh"), (b,), dy)
    w2 = w.clone().requires_grad_(True)
    both = torch.autograd.grad(mpe_hip.linear(x, w2, b, "tanh"), (w2, b), dy)
    z, size, _ = forward64(x, w, b.detach(), None, "tanh")
    d = dy.double()
    want = (d * slope64(z, "tanh")).sum(0)
    e = d.abs() * (0.9 * (k + 8) * V * size + 16 * V * (1 + z.abs()))
    bound = (e.sum(0) + (m + 8) * V * (d * slope64(z, "tanh")).abs().sum(0)) * (1 + U[dt]) + U[dt] * want.abs() + TINY[dt]
    inside(db, want, bound, "db")
    inside(both[1], want, bound, "db beside dw")


@pytest.mark.parametrize("k", [1024, 1000])
def test_large_tiles_give_the_same_every_time(k):
    """A stage of LDS that is overwritten before every wave has read it shows in a few elements of a few runs."""
    import mpe_hip
    m, n = 32768, 1024
    x, w, b, r, dy = make(m, k, n, torch.bfloat16, residual=True)
    q = [t.requires_grad_(True) for t in (x, w, b)]
    first = None
    for _ in range(24):
        y = mpe_hip.linear(*q, "gelu", r)
        got = (y.detach(),) + torch.autograd.grad(y, q, dy)
        first = first or got
        assert all(torch.equal(a, c) for a, c in zip(got, first))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ACTS)
def test_every_activation_in_large_tiles(act, dt):
    x, w, b, r, dy = make(8193, 96, 1028, dt, residual=True, exact=act == "relu")
    check_forward(x, w, b, r, act)
    check_forward(x, w, None, None, act)
    check_backward(x, w, b, r, dy, act)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [65, 67, 70, 71, 88, 95])
def test_large_sums_that_end_where_memory_ends(k, dt):
    """Copies to LDS at the end of the sum, every kind of last chunk: the last row ends with its buffer, NaN behind it and in
    the gap between the rows."""
    import mpe_hip
    m, n, ld = 16400, 520, k + (k & 1)
    x, w, b, r, dy = make(m, k, n, dt, residual=True)
    def framed(t):
        flat = torch.full(((t.shape[0] + 1) * ld + 64,), math.nan, device=DEV).to(dt)
        v = flat[34:34 + t.shape[0] * ld].view(t.shape[0], ld)[:, :t.shape[1]]
        v.copy_(t)
        return v
    one, two = mpe_hip.linear(x, w, b, "silu", r), mpe_hip.linear(framed(x), framed(w), b, "silu", r)
    check_forward(framed(x), framed(w), b, r, "silu")
    assert k & 1 or torch.equal(one, two)           # an odd row stride goes another way


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_one_upstream_row_for_all_in_large_tiles(dt):
    """dy expanded over the rows, its end inside a chunk and at the end of its memory."""
    import mpe_hip
    m, k, n = 65537, 128, 270
    x, w, b, _, _ = make(m, k, n, dt)
    row = torch.full((2 * n + 64,), math.nan, device=DEV).to(dt)[32:32 + n].copy_(torch.randn(n, device=DEV).to(dt))
    q = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    y = mpe_hip.linear(*q)
    got = torch.autograd.grad(y, q, row.expand(m, n))
    want = torch.autograd.grad(mpe_hip.linear(*q), q, row.expand(m, n).contiguous())
    assert torch.equal(got[0], want[0])
    # two orders of m float32 additions, then one rounding each
    mags = (row.double().abs()[:, None] * x.double().abs().sum(0), m * row.double().abs())
    for a, c, mag in zip(got[1:], want[1:], mags):
        fits = mag < torch.finfo(dt).max / 2 if dt == torch.float16 else torch.ones_like(mag, dtype=torch.bool)       # 65537 equal numbers pass float16's range: sums of them have to do so both times
        assert torch.equal(a[~fits].isinf(), c[~fits].isinf())
        inside(a[fits], c[fits].double(), (2 * (m + 8) * V * mag + 2 * U[dt] * c.double().abs() + TINY[dt])[fits], "two orders")


def test_more_rows_than_a_grid_dimension_of_strips():
    """Column sums over 8.4 M rows.  Values of -1, 0 and 1: every sum stays below 2^24 and is exact in float32."""
    import mpe_hip
    period, times = 1024, 8204
    g = torch.Generator(DEV).manual_seed(5)
    xp, dp = (torch.randint(-1, 2, (period, c), device=DEV, generator=g).to(torch.bfloat16) for c in (256, 128))
    w, b = torch.zeros(128, 256, device=DEV, dtype=torch.bfloat16).requires_grad_(True), torch.zeros(128, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    dw, db = torch.autograd.grad(mpe_hip.linear(xp.repeat(times, 1), w, b), (w, b), dp.repeat(times, 1))
    assert torch.equal(dw, (dp.double().T @ xp.double() * times).to(torch.bfloat16))
    assert torch.equal(db, (dp.double().sum(0) * times).to(torch.bfloat16))


@pytest.mark.parametrize("dt", DTYPES)
def test_long_reduction_over_rows(dt):
    """The weight gradient of a whole rollout step: many rows, few columns."""
    x, w, b, r, dy = make(70001, 14, 9, dt)
    check_backward(x, w, b, r, dy, "tanh")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("ld,k", [(42, 14), (43, 14), (100, 33), (75, 75)])
def test_strided_rows_and_odd_offsets(dt, ld, k):
    """One agent's columns of everybody's observations; the view starts at an odd element where ld - k is odd."""
    x, w, b, r, dy = make(300, k, 40, dt, ld=ld)
    check_forward(x, w, b, r, "tanh")
    check_backward(x, w, b, r, dy, "tanh")
    wide = torch.randn(80, k + 3, device=DEV).to(dt)[::2, 1:k + 1]       # weight rows strided as well
    check_forward(x, wide, b, None, "silu")
    check_backward(x, wide, b, None, dy, "silu")


def test_views_of_the_environment_go_in_as_they_lie():
    import mpe_hip
    env = mpe_hip.BatchedEnv("simple_tag", 333, device=DEV)
    env.reset(seed=3)
    for i, obs in enumerate(env.obs_n):
        w = torch.randn(24, obs.shape[1], device=DEV) * 0.2
        check_forward(obs, w, None, None, "tanh")
    three = torch.randn(7, 5, 6, device=DEV)
    w, b = torch.randn(4, 6, device=DEV), torch.randn(4, device=DEV)
    got = mpe_hip.linear(three, w, b)
    assert got.shape == (7, 5, 4) and torch.equal(got.view(35, 4), mpe_hip.linear(three.view(35, 6), w, b))
    assert torch.equal(mpe_hip.linear(three[0, 0], w, b), mpe_hip.linear(three[0, :1], w, b)[0])
    turned = torch.randn(6, 35, device=DEV).T                               # columns contiguous: copied
    assert torch.equal(mpe_hip.linear(turned, w, b), mpe_hip.linear(turned.contiguous(), w, b))


def test_expanded_residual_and_upstream_gradient():
    """A broadcast residual is read with row stride 0 and its gradient is summed; so is a gradient that sum() expands."""
    import mpe_hip
    x, w, b, _, dy = make(50, 20, 12, torch.float32)
    row = torch.randn(12, device=DEV, requires_grad=True)
    y = mpe_hip.linear(x, w, b, activation="tanh", residual=row.expand(50, 12))
    z, size, want = forward64(x, w, b, row.detach().expand(50, 12), "tanh")
    inside(y.detach(), want, forward_bound(z, size, want, row.detach().expand(50, 12), "tanh", 20, torch.float32), "y")
    (g,) = torch.autograd.grad(y, row, dy)
    inside(g, dy.double().sum(0), 60 * V * dy.double().abs().sum(0), "residual row")
    x1, w1 = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    one = torch.autograd.grad(mpe_hip.linear(x1, w1, b, activation="gelu").sum(), (x1, w1))
    two = torch.autograd.grad(mpe_hip.linear(x1, w1, b, activation="gelu"), (x1, w1), torch.ones(50, 12, device=DEV))
    assert all(torch.equal(p, q) for p, q in zip(one, two))
    # sliced and transposed upstream gradients
    wide = torch.randn(50, 30, device=DEV)
    got = torch.autograd.grad(mpe_hip.linear(x1, w1, b, activation="gelu"), (x1, w1), wide[:, 5:17])
    want = torch.autograd.grad(mpe_hip.linear(x1, w1, b, activation="gelu"), (x1, w1), wide[:, 5:17].contiguous())
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    got = torch.autograd.grad(mpe_hip.linear(x1, w1, b), (x1, w1), torch.randn(12, 50, device=DEV).T)
    assert got[0].shape == (50, 20)


def test_only_what_is_asked_for_is_computed():
    import mpe_hip
    x, w, b, r, dy = make(33, 10, 7, torch.float32, residual=True)
    for need in range(1, 16):
        ts = [t.detach().requires_grad_(bool(need >> i & 1)) for i, t in enumerate((x, w, b, r))]
        y = mpe_hip.linear(ts[0], ts[1], ts[2], activation="tanh", residual=ts[3])
        got = torch.autograd.grad(y, [t for t in ts if t.requires_grad], dy)
        full = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        want = torch.autograd.grad(mpe_hip.linear(full[0], full[1], full[2], activation="tanh", residual=full[3]), full, dy)
        for g, i in zip(got, [i for i in range(4) if need >> i & 1]):
            assert torch.equal(g, want[i])
    with torch.no_grad():
        assert not mpe_hip.linear(*[t.detach().requires_grad_(True) for t in (x, w, b)]).requires_grad


def test_no_rows():
    import mpe_hip
    w, b = torch.randn(6, 5, device=DEV, requires_grad=True), torch.randn(6, device=DEV, requires_grad=True)
    x = torch.zeros(0, 5, device=DEV, requires_grad=True)
    y = mpe_hip.linear(x, w, b, activation="tanh")
    assert y.shape == (0, 6)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros(0, 6, device=DEV))
    assert dx.shape == (0, 5) and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros_like(b))


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("m,k,n", [(40, 70, 90), (7, 200, 33), (300, 128, 64)])
def test_infinities_and_nan_stay_in_their_rows(dt, m, k, n):
    import mpe_hip
    x, w, b, _, _ = make(m, k, n, dt)
    clean = mpe_hip.linear(x, w, b)
    x2 = x.clone()
    x2[1, 3], x2[2, k - 1], x2[5, 0], x2[5, 1], x2[6, k // 2] = math.inf, -math.inf, math.inf, -math.inf, math.nan
    w2 = w.clone()
    w2[:, 3], w2[:, k - 1] = w2[:, 3].abs() + 0.5, w2[:, k - 1].abs() + 0.5       # a sign that every infinity keeps
    w2[4, 3] = 0.0                                                                  # inf * 0
    got, want = mpe_hip.linear(x2, w2, b), (x2.double() @ w2.double().T + b.double())
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf].double(), want[inf])
    rows = [i for i in range(m) if i not in (1, 2, 5, 6)]
    assert torch.equal(got[rows], mpe_hip.linear(x, w2, b)[rows]) and not torch.isnan(clean).any()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("k", [12, 40, 96])
def test_gradients_of_infinite_inputs_and_weights_are_infinite(k, dt):
    """One infinity in x or w: where it meets a dz that is not zero the gradient is infinite, not NaN, and elsewhere finite."""
    import mpe_hip
    m, n = 70, 24
    x, w, b, _, dy = make(m, k, n, dt)
    dy = dy.abs() + 0.5                                  # exact in no type's second piece, never zero
    dy[:, ::2] *= -1
    w = w.abs() + 0.25
    x = x.abs() + 0.25
    for t, at in ((x, (3, 2)), (w, (1, 0))):
        q = [x.clone(), w.clone()]
        q[0 if t is x else 1][at] = math.inf
        q = [t.requires_grad_(True) for t in q]
        dx, dw = torch.autograd.grad(mpe_hip.linear(q[0], q[1], None, "relu"), q, dy)
        if t is x:
            assert torch.equal(dw[:, 2].float(), torch.copysign(torch.full((n,), math.inf, device=DEV), dy[3].float()))
            keep = [c for c in range(k) if c != 2]
            assert torch.isfinite(dx).all() and torch.isfinite(dw[:, keep]).all()
        else:
            assert torch.equal(dx[:, 0].float(), torch.copysign(torch.full((m,), math.inf, device=DEV), dy[:, 1].float()))
            assert torch.isfinite(dw).all() and torch.isfinite(dx[:, 1:]).all()


def test_float32_extremes():
    """The largest and the smallest float32 go through products and come out as float32 would have them."""
    import mpe_hip
    big = torch.finfo(torch.float32).max
    for m in (3, 100):
        x = torch.zeros(m, 40, device=DEV)
        x[0, 0], x[1, 1], x[2, 2] = big, 2.0 ** -120, -big
        x[3 % m, 5] = 1.0
        w = torch.zeros(70, 40, device=DEV)
        w[:, 0], w[:, 1], w[:, 2], w[1, 0] = 1.0, 0.75, 0.5, 2.0
        y = mpe_hip.linear(x, w)
        assert float(y[0, 0]) == big and float(y[0, 1]) == math.inf and float(y[1, 0]) == 0.75 * 2.0 ** -120 and float(y[2, 0]) == -big * 0.5


@pytest.mark.parametrize("act", ["tanh", "gelu", "silu", "none"])
def test_gradient_against_differences(act):
    """<grad, d> against (f(+h) - f(-h)) / 2h of the kernels' own forward, f = <y, dy> summed in float64, h = 2^-6: the third
    derivatives of these activations stay below 6, so the difference is off by h^2 / 6 * 6 * sum |dy| |dz.d|^3, and by the
    rounding of y, 2 (K + 16) 2^-24 per unit of sum |dy| (|x||w| + 1) / 2h."""
    import mpe_hip
    m, k, n = 20, 12, 10
    x, w, b, r, dy = [t.detach() for t in make(m, k, n, torch.float32, residual=True)]
    g = torch.Generator(DEV).manual_seed(5)
    h = 2.0 ** -6
    for i, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, device=DEV, generator=g)
        f = lambda s: (mpe_hip.linear(*[q + s * h * d if j == i else q for j, q in enumerate((x, w, b))], activation=act, residual=r).double() * dy.double()).sum()
        leaf = t.clone().requires_grad_(True)
        y = mpe_hip.linear(*[leaf if j == i else q for j, q in enumerate((x, w, b))], activation=act, residual=r)
        (grad,) = torch.autograd.grad(y, leaf, dy)
        move = (d.double() @ w.double().T if i == 0 else x.double() @ d.double().T if i == 1 else d.double().expand(m, n)).abs()
        size = x.double().abs() @ w.double().abs().T + b.double().abs() + r.double().abs() + h * move + 1
        bound = h * h * (dy.double().abs() * move ** 3).sum() + (dy.double().abs() * size).sum() * 2 * (k + 16) * V / (2 * h)
        assert abs(float((f(1) - f(-1)) / (2 * h)) - float((grad.double() * d.double()).sum())) <= float(bound)


def test_results_do_not_change_from_run_to_run():
    import mpe_hip
    for m, k, n, dt in ((30011, 66, 65, torch.float32), (5000, 300, 200, torch.bfloat16), (9, 512, 300, torch.float32)):
        x, w, b, r, dy = make(m, k, n, dt)
        out = []
        for _ in range(3):
            ls = [t.detach().requires_grad_(True) for t in (x, w, b)]
            y = mpe_hip.linear(*ls, activation="gelu")
            out.append([y.detach()] + list(torch.autograd.grad(y, ls, dy)))
            torch.empty(1 << 22, device=DEV).normal_()
        assert all(torch.equal(p, q) for o in out[1:] for p, q in zip(out[0], o))


def test_captured_forward_and_backward_replay():
    """One capture of forward and gradients, replayed between eager work on new inputs in the same buffers."""
    import mpe_hip
    for m, k, n, dt in ((3000, 64, 64, torch.float32), (3, 14, 64, torch.float32), (700, 200, 136, torch.bfloat16)):
        x, w, b, r, dy = make(m, k, n, dt, residual=True)
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b, r)]
        call = lambda ls: (lambda y: [y.detach()] + list(torch.autograd.grad(y, ls, dy)))(mpe_hip.linear(ls[0], ls[1], ls[2], activation="silu", residual=ls[3]))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(leaves)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(leaves)
        for i in range(3):
            with torch.no_grad():
                for t in leaves:
                    t.copy_(torch.randn_like(t))
                dy.copy_(torch.randn_like(dy))
            graph.replay()
            torch.cuda.synchronize()
            want = call([t.detach().clone().requires_grad_(True) for t in leaves])
            assert all(torch.equal(p, q) for p, q in zip(out, want)), (m, k, n, i)
            torch.cuda.synchronize()


def test_on_another_stream_and_two_calls_at_once():
    import mpe_hip
    x, w, b, r, dy = make(20000, 64, 64, torch.float32)
    want = mpe_hip.linear(x, w, b, activation="tanh")
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ls = [t.detach().requires_grad_(True) for t in (x, w, b)]
            y = mpe_hip.linear(*ls, activation="tanh")
            outs.append([y.detach()] + list(torch.autograd.grad(y, ls, dy)))
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], want) and all(torch.equal(p, q) for p, q in zip(*outs))


def test_saved_inputs_may_not_be_written_before_the_backward_pass():
    import mpe_hip
    x, w, b, r, dy = make(10, 5, 4, torch.float32)
    w1 = w.detach().clone().requires_grad_(True)
    y = mpe_hip.linear(x, w1, b, activation="tanh")
    with torch.no_grad():
        w1.mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(y, w1, dy)


def test_refusals():
    import mpe_hip
    x, w, b = torch.zeros(4, 3, device=DEV), torch.zeros(2, 3, device=DEV), torch.zeros(2, device=DEV)
    for args, kw in (((x.double(), w.double()), {}), ((x, w.bfloat16()), {}), ((x, w[:, :2]), {}), ((x, w, b[:1]), {}), ((x, w.cpu()), {}),
                     ((x, w, b), dict(residual=torch.zeros(4, 3, device=DEV))), ((x, w, b), dict(residual=torch.zeros(1, 2, device=DEV))),
                     ((x[:, :0], w[:, :0]), {}), ((x, w[:0]), {}), ((torch.zeros((), device=DEV), w), {}), ((x, w, b.bfloat16()), {})):
        with pytest.raises(ValueError):
            mpe_hip.linear(*args, **kw)
    lx = x.requires_grad_(True)
    (g,) = torch.autograd.grad(mpe_hip.linear(lx, w, activation="tanh").sum(), lx, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), lx)
