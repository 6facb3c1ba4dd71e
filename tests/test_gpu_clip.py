"""Global norm and clipping against float64.  The squares are summed in float64, so the norm is the float64 one rounded to
float32 (2^-24, and a few 2^-53 per element of the sum); a clipped element is one float32 product by a factor that was rounded
once, then rounded to its type: (3 * 2^-24 + u) |value|."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def tensors(sizes, dts, seed=0, spread=1.0):
    g = torch.Generator(DEV).manual_seed(seed)
    return [(spread * torch.randn(s, device=DEV, generator=g)).to(dts[i % len(dts)]) for i, s in enumerate(sizes)]


def norm64(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def check(ts, max_norm, outs, norm):
    want = norm64(ts)
    assert norm.dtype == torch.float32 and norm.dim() == 0
    assert abs(float(norm) - want) <= 2.0 ** -23 * want
    f = max_norm / want if want > max_norm else 1.0
    for t, o in zip(ts, outs):
        ref = t.double() * f
        if f == 1.0:
            assert torch.equal(o, t)
        else:
            assert ((o.double() - ref).abs() <= (3 * 2.0 ** -24 + U[t.dtype]) * ref.abs() * (1 + 2.0 ** -20) + TINY[t.dtype]).all()


SETS = [[1], [3, 1, 2], [64, 896, 64, 4096, 5], [255, 256, 257, 8191, 8192, 8193], [100003], [0, 5, 0, 17], [7] * 300, [1 << 22, 3, 1 << 20]]


@pytest.mark.parametrize("dts", [(torch.float32,), (torch.bfloat16,), (torch.float16,), (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: "%d_tensors_%d" % (len(s), sum(s)))
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_clip(sizes, dts, max_norm):
    import mpe_hip
    ts = tensors(sizes, dts, spread=0.3)
    outs = [torch.full_like(t, 9.0) for t in ts]
    norm = mpe_hip.clip_grad_norm(ts, max_norm, out=outs)
    check(ts, max_norm, outs, norm)
    assert torch.equal(mpe_hip.grad_norm(ts), norm)
    params = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts] + [torch.nn.Parameter(torch.zeros(3, device=DEV))]
    for p, t in zip(params, ts):
        p.grad = t.clone()
    assert torch.equal(mpe_hip.clip_grad_norm_(params, max_norm), norm) and params[-1].grad is None
    assert all(torch.equal(p.grad, o) for p, o in zip(params, outs))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_neighbours_of_odd_slices_stay_as_they_were(dt):
    """Slices of one buffer at every offset: what lies between and behind them is not written."""
    import mpe_hip
    flat = torch.randn(60000, device=DEV).to(dt)
    spans = [(1, 2), (3, 4), (7, 1000), (1001, 1002), (1003, 20000), (20005, 45678)]
    src = [torch.randn(b - a, device=DEV).to(dt) for a, b in spans]
    before = flat.clone()
    outs = [flat[a:b] for a, b in spans]
    norm = mpe_hip.clip_grad_norm(src, 0.25, out=outs)
    check(src, 0.25, outs, norm)
    keep = torch.ones(60000, dtype=torch.bool, device=DEV)
    for a, b in spans:
        keep[a:b] = False
    assert torch.equal(flat[keep], before[keep])
    mid = [before[a:b].clone() for a, b in spans]       # odd slices as sources, in place
    odd = before.clone()
    mpe_hip.clip_grad_norm([odd[a:b] for a, b in spans], 0.5, out=[odd[a:b] for a, b in spans])
    even = [t.clone() for t in mid]
    mpe_hip.clip_grad_norm(mid, 0.5, out=even)
    assert all(torch.equal(odd[a:b], t) for (a, b), t in zip(spans, even)) and torch.equal(odd[keep], before[keep])


def test_extreme_values():
    import mpe_hip
    big = torch.full((1000,), 3e38, device=DEV)
    out = [torch.empty_like(big)]
    norm = mpe_hip.clip_grad_norm([big], 1.0, out=out)
    assert math.isinf(float(norm))                      # 9.5e39 is beyond float32, and still no NaN in the factor
    check_ref = 1.0 / (3e38 * math.sqrt(1000))
    assert torch.allclose(out[0].double(), big.double() * check_ref, rtol=1e-6, atol=0)
    small = torch.full((1000,), 1e-30, device=DEV)
    assert abs(float(mpe_hip.grad_norm([small])) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    zero = torch.zeros(5, device=DEV)
    assert float(mpe_hip.clip_grad_norm([zero], 0.0, out=[zero])) == 0.0 and torch.equal(zero, torch.zeros(5, device=DEV))
    one = torch.ones(4, device=DEV)
    assert float(mpe_hip.clip_grad_norm([one], 0.0, out=[one])) == 2.0 and torch.equal(one, torch.zeros(4, device=DEV))
    a, b = torch.tensor([1.0, math.inf], device=DEV), torch.ones(3, device=DEV)
    norm = mpe_hip.clip_grad_norm([a, b], 1.0, out=[a, b])
    assert math.isinf(float(norm)) and float(a[0]) == 0 and math.isnan(float(a[1])) and torch.equal(b, torch.zeros(3, device=DEV))
    a, b = torch.tensor([1.0, math.nan], device=DEV), torch.ones(3, device=DEV)
    assert math.isnan(float(mpe_hip.clip_grad_norm([a, b], 1.0, out=[a, b]))) and torch.isnan(a).all() and torch.isnan(b).all()


def test_orders_of_dimensions():
    import mpe_hip
    t = torch.randn(30, 40, device=DEV).T
    c = torch.randn(4, 5, 6, device=DEV).permute(2, 0, 1)
    want = [t.contiguous().clone(), c.contiguous().clone()]
    mpe_hip.clip_grad_norm(want, 0.1, out=want)
    mpe_hip.clip_grad_norm([t, c], 0.1, out=[t, c])
    # the order of the sum follows memory, so the factor may differ in its last bit
    assert torch.allclose(t, want[0], rtol=1e-6, atol=0) and torch.allclose(c, want[1], rtol=1e-6, atol=0)


def test_repeat_capture_and_streams():
    import mpe_hip
    for sizes in (SETS[2], SETS[7]):
        ts = tensors(sizes, (torch.float32, torch.bfloat16))
        outs = [torch.empty_like(t) for t in ts]
        norm = mpe_hip.clip_grad_norm(ts, 0.5, out=outs)
        for _ in range(3):
            again = [torch.empty_like(t) for t in ts]
            assert torch.equal(mpe_hip.clip_grad_norm(ts, 0.5, out=again), norm) and all(torch.equal(p, q) for p, q in zip(outs, again))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = mpe_hip.clip_grad_norm(ts, 0.5, out=outs)
        for i in range(3):
            for t in ts:
                t.copy_(torch.randn_like(t))
            graph.replay()
            torch.cuda.synchronize()
            fresh = [torch.empty_like(t) for t in ts]
            assert torch.equal(mpe_hip.clip_grad_norm(ts, 0.5, out=fresh), held) and all(torch.equal(p, q) for p, q in zip(outs, fresh))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = [torch.empty_like(t) for t in ts]
            n2 = mpe_hip.clip_grad_norm(ts, 0.5, out=there)
        side.synchronize()
        assert torch.equal(n2, held) and all(torch.equal(p, q) for p, q in zip(there, outs))


def test_refusals():
    import mpe_hip
    t = torch.zeros(4, 6, device=DEV)
    for ts, out in (([t.double()], [t.double()]), ([t[:, ::2]], [t[:, ::2]]), ([t, t], [t, t]), ([t, t.clone()], [t, t]), ([t], [t.half()]), ([t], [t.T]),
                    ([t[:1].expand(4, 6)], [t]), ([t], [t[:2]]), ([t, t.cpu()], [t, t.clone()]), ([t.to_sparse()], [t]),
                    ([t, torch.zeros(24, device=DEV)], [t, t.view(24)])):
        with pytest.raises(ValueError):
            mpe_hip.clip_grad_norm(ts, 1.0, out=out)
    buf = torch.zeros(40, device=DEV)
    with pytest.raises(mpe_hip.MpeError):
        mpe_hip.clip_grad_norm([buf[:30]], 1.0, out=[buf[10:]])
    p = torch.nn.Parameter(t.clone())
    q = (p * p).sum()
    with torch.no_grad():
        mpe_hip.clip_grad_norm([p], 1.0, out=[p])           # written in place: autograd is told
    with pytest.raises(RuntimeError, match="modified"):
        q.backward()


def test_destinations_that_meet_other_sources_or_carry_gradients_are_refused():
    import mpe_hip
    a, b = torch.ones(8, device=DEV), torch.ones(8, device=DEV)
    with pytest.raises(mpe_hip.MpeError, match="overlaps the source"):
        mpe_hip.clip_grad_norm([a, b], 1.0, out=[b, a])
    p = torch.ones(8, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="requires gradients"):
        mpe_hip.clip_grad_norm([a], 1.0, out=[p])
    with torch.no_grad():
        mpe_hip.clip_grad_norm([a], 1.0, out=[p])
    assert torch.allclose(p.detach(), torch.full_like(a, 8 ** -0.5), rtol=2.0 ** -23, atol=0)
    # a source may be given twice, with two destinations
    c, d = torch.empty_like(a), torch.empty_like(a)
    norm = mpe_hip.clip_grad_norm([a, a], 2.0, out=[c, d])
    assert float(norm) == 4.0 and torch.equal(c, torch.full_like(a, 0.5)) and torch.equal(d, c)
