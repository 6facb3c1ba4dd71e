"""mpe_hip.ppo_loss against float64.  Bounds, with v = 2^-24: a log-probability is a difference of float32 numbers, off by
8 v (|l - max| + |log sum| + |old| + 1); the ratio carries that relatively; sums over rows are in float64.  A logit's gradient
is off by 32 v times the sum of its two parts' sizes and their relative error, and is rounded once to the type."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
V = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def make(rows, v, dt=torch.float32, values=True, mask=None, weights=False, seed=0, i64=False):
    g = torch.Generator(DEV).manual_seed(seed + 31 * rows + v)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
    logits = (1.5 * rnd(rows, v)).to(dt)
    d = dict(logits=logits, actions=torch.randint(0, v, (rows,), device=DEV, generator=g, dtype=torch.int64 if i64 else torch.int32))
    allowed = None
    if mask:
        allowed = torch.rand(rows, v, device=DEV, generator=g) < 0.6
        allowed[::7] = False                        # nothing left
        allowed[1::7].scatter_(1, d["actions"][1::7, None].long(), True)
    lp = torch.log_softmax(logits.double(), 1).gather(1, d["actions"].long()[:, None])[:, 0]
    lr = 0.3 * rnd(rows).double()
    for border in (0.8, 1.2):                      # clear of the borders, where the last bit would choose the branch
        lr = torch.where((lr.exp() - border).abs() < 1e-2, lr + 0.05, lr)
    if allowed is not None:
        lm = logits.double().masked_fill(~allowed, -math.inf)
        lp2 = lm.gather(1, d["actions"].long()[:, None])[:, 0] - torch.logsumexp(lm, 1)
        lp = torch.where(torch.isfinite(lp2), lp2, lp)
    d.update(old_logp=(lp - lr).float(), advantages=rnd(rows), action_mask=allowed)
    if values:
        d["old_values"] = rnd(rows)
        d["values"], d["returns"] = d["old_values"] + 0.3 * rnd(rows), d["old_values"] + rnd(rows)
    if weights:
        d["weights"] = torch.rand(rows, device=DEV, generator=g) * (torch.rand(rows, device=DEV, generator=g) < 0.7)
    return d


def reference(d, clip=0.2, value_clip=None, value_coef=0.5, entropy_coef=0.01):
    """Loss, stats, gradients in float64, by differentiating the formula; and each row's share."""
    v = d["logits"].shape[-1]
    l = d["logits"].detach().double().reshape(-1, v).requires_grad_(True)
    f = lambda k: None if d.get(k) is None else d[k].detach().reshape(-1).double()
    act, w = d["actions"].reshape(-1).long(), f("weights")
    w = torch.ones(l.shape[0], dtype=torch.float64, device=DEV) if w is None else w
    ok = torch.ones_like(l, dtype=torch.bool) if d.get("action_mask") is None else d["action_mask"].reshape(-1, v).bool()
    ok = ok & (l.detach() != -math.inf)
    live = (w != 0) & (act >= 0) & (act < v) & ok.gather(1, act.clamp(0, v - 1)[:, None])[:, 0]
    w = torch.where(live, w, torch.zeros_like(w))
    share = w / w.sum() if live.any() else w
    safe_act = act.clamp(0, v - 1)
    sc = torch.where(live[:, None], l, torch.zeros_like(l)).masked_fill(live[:, None] & ~ok, -math.inf)
    logp = torch.log_softmax(sc, 1)
    lpz = torch.where(logp == -math.inf, torch.zeros_like(logp), logp)
    ent = -(logp.exp() * lpz).sum(1)
    at = logp.gather(1, safe_act[:, None])[:, 0]
    old, adv = torch.where(live, f("old_logp"), at.detach()), torch.where(live, f("advantages"), torch.zeros_like(w))
    q = (at - old).exp()
    pg = -torch.minimum(q * adv, q.clamp(1 - clip, 1 + clip) * adv)
    value, val = torch.zeros((), dtype=torch.float64, device=DEV), f("values")
    if val is not None:
        val.requires_grad_(True)
        mine, o, r = [torch.where(live, t, torch.zeros_like(w)) for t in (val, f("old_values"), f("returns"))]
        u = (mine - r) ** 2
        if value_clip is not None:
            u = torch.maximum(u, (o + (mine - o).clamp(-value_clip, value_clip) - r) ** 2)
        value = 0.5 * (share * u).sum()
    pol, en = (share * pg).sum(), (share * torch.where(live, ent, torch.zeros_like(ent))).sum()
    loss = pol + value_coef * value - entropy_coef * en
    kl = (share * torch.where(live, 0.5 * (at - old) ** 2, torch.zeros_like(w))).sum()
    stats = torch.stack([pol, value, en, kl, (share * ((q - 1).abs() > clip) * live).sum()]).detach()
    grads = torch.autograd.grad(loss, [l] + ([val] if val is not None else []))
    size = dict(q=q.detach(), adv=adv, share=share, logp=lpz.detach(), p=logp.detach().exp(), ent=ent.detach(), at=at.detach(), old=old)
    return loss.detach(), stats, grads, size


def check(d, **kw):
    import mpe_hip
    leaves = [d[k].requires_grad_(True) for k in ("logits", "values") if d.get(k) is not None]
    loss, stats = mpe_hip.ppo_loss(**d, **kw)
    got = torch.autograd.grad(loss, leaves)
    want_loss, want_stats, grads, s = reference(d, **kw)
    dt = d["logits"].dtype
    lse = (s["logp"].abs().amax(1) + 1)
    rel = 8 * V * (lse + s["old"].abs() + s["at"].abs().clamp(max=1e4) + 1)                    # of the ratio
    e = (s["share"].abs() * (s["q"] * s["adv"].abs() + 1 + lse * lse + s["old"].abs())).sum()
    big = float((s["share"].abs() * rel * (s["q"] * s["adv"].abs() + 1 + (s["at"] - s["old"]).abs())).sum() + 32 * V * e)
    assert loss.dtype == torch.float32 and loss.dim() == 0 and stats.shape == (5,)
    for i in range(5):
        assert abs(float(stats[i]) - float(want_stats[i])) <= big + 4 * V * abs(float(want_stats[i])), (i, float(stats[i]), float(want_stats[i]))
    assert abs(float(loss.detach()) - float(want_loss)) <= 2 * big
    ce = abs(kw.get("entropy_coef", 0.01))
    g1 = (s["share"] * s["q"] * s["adv"]).abs()[:, None]
    hot = torch.nn.functional.one_hot(d["actions"].reshape(-1).long().clamp(0, d["logits"].shape[-1] - 1), d["logits"].shape[-1]).double()
    pol, en = g1 * (hot + s["p"]), ce * s["share"].abs()[:, None] * s["p"] * (s["logp"].abs() + s["ent"].abs()[:, None])
    rel_p = 8 * V * (s["logp"].abs() + lse[:, None] + 1)
    off = pol * (rel[:, None] + rel_p + 32 * V) + en * (rel_p + 32 * V) + ce * s["share"].abs()[:, None] * s["p"] * rel_p
    ref = grads[0]
    gl = got[0].reshape(ref.shape).double()
    bad = ~((gl - ref).abs() <= off + U[dt] * (ref.abs() + off) + TINY[dt])
    assert not bad.any(), "dlogits: %d of %d outside" % (int(bad.sum()), bad.numel())
    if len(got) > 1:
        assert ((got[1].reshape(-1).double() - grads[1]).abs() <= 16 * V * grads[1].abs() + TINY[torch.float32]).all()
    return loss.detach(), stats, got


SIZES = [(1, 1), (1, 5), (75, 5), (64, 2), (1000, 5), (333, 7), (257, 8), (300, 9), (129, 16), (200, 17), (50, 31), (60, 64), (33, 65), (40, 100), (17, 255), (10, 256),
         (9, 513), (5, 1000), (3, 2049), (2, 8192), (2, 20011), (70000, 5), (20000, 3), (4100, 33)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", SIZES)
def test_against_the_formula(rows, v, dt):
    i = SIZES.index((rows, v))
    check(make(rows, v, dt, values=i % 2 == 0, mask=i % 3 == 1, weights=i % 4 == 3, i64=i % 5 == 2), value_clip=0.2 if i % 4 < 2 else None)


@pytest.mark.parametrize("rows,v", [(100, 5), (90, 40), (30, 700), (6, 9000)])
def test_masks_weights_and_value_clipping_together(rows, v):
    for mask in (False, True):
        for weights in (False, True):
            check(make(rows, v, mask=mask, weights=weights), value_clip=0.15, value_coef=0.7, entropy_coef=0.3, clip=0.2)


@pytest.mark.parametrize("rows,v", [(40, 5), (40, 70), (12, 3000)])
def test_rows_that_are_left_out(rows, v):
    """Weight 0, an action outside the moves, nothing allowed, every logit -infinity: zero gradients, and what such a row holds
    (NaN, infinities) reaches nothing."""
    import mpe_hip
    d = make(rows, v, mask=True, weights=True)
    d["weights"] = torch.ones(rows, device=DEV)
    d["action_mask"][0] = False
    d["logits"][1] = -math.inf
    d["actions"][2], d["actions"][3], d["weights"][4] = -1, v, 0.0
    for i in (0, 2, 3, 4):
        d["logits"][i] = math.nan
    for k in ("old_logp", "advantages", "values", "returns"):
        d[k][:5] = math.nan
    out = torch.arange(rows, device=DEV) < 5
    loss, stats, got = check(d, value_clip=0.2)
    assert not torch.isnan(loss) and not torch.isnan(stats).any()
    assert torch.equal(got[0][out], torch.zeros_like(got[0][out])) and torch.equal(got[1][out], torch.zeros(5, device=DEV))
    keep = {k: (t[~out].detach() if t is not None else None) for k, t in d.items()}
    alone = mpe_hip.ppo_loss(**keep, value_clip=0.2)
    assert torch.allclose(loss, alone[0], rtol=1e-6, atol=1e-7)
    d["weights"] = torch.zeros(rows, device=DEV)
    loss, stats = mpe_hip.ppo_loss(**d)
    g = torch.autograd.grad(loss, d["logits"])[0]
    assert float(loss.detach()) == 0 and torch.equal(stats, torch.zeros(5, device=DEV)) and torch.equal(g, torch.zeros_like(g))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [6, 50, 5000])
def test_lowest_values_infinities_and_nan_in_masked_places(v, dt):
    import mpe_hip
    rows = 24
    d = make(rows, v, dt, mask=True)
    d["action_mask"] = torch.ones(rows, v, dtype=torch.bool, device=DEV)
    d["actions"].fill_(0)
    d["action_mask"][:, 1:4] = False
    d["logits"][:, 1], d["logits"][:, 2], d["logits"][:, 3] = math.nan, math.inf, -math.inf
    base = check(d)
    d2 = dict(d, logits=d["logits"].detach().clone())
    d2["logits"][:, 1:4] = 0.0
    again = check(d2)
    assert torch.equal(base[0], again[0]) and torch.equal(base[2][0], again[2][0])
    # masks written into the logits: the type's lowest value and -infinity
    low = dict(d2, logits=d2["logits"].detach().clone(), action_mask=None)
    low["logits"][:, 1], low["logits"][:, 2], low["logits"][:, 3] = torch.finfo(dt).min, -math.inf, torch.finfo(dt).min
    third = check(low)
    if dt != torch.float16:                         # exp(-65504) is 0 too: the three agree in every type
        assert torch.equal(third[0], base[0])
    allow = dict(low, logits=torch.full((rows, v), torch.finfo(dt).min, dtype=dt, device=DEV))
    loss, stats = mpe_hip.ppo_loss(**allow)         # every logit the lowest: a uniform choice
    assert abs(float(stats[2]) - math.log(v)) < 1e-5
    nan = dict(d2, logits=d2["logits"].detach().clone())
    nan["logits"][3] = math.nan                     # where it is allowed it has to show
    assert math.isnan(float(mpe_hip.ppo_loss(**nan)[0]))


def test_shapes_strides_and_types():
    import mpe_hip
    T, B, A, v = 4, 6, 3, 5
    d = make(T * B * A, v)
    flat = check(d)
    cube = {k: (None if t is None else t.detach().view((T, B, A) + t.shape[1:])) for k, t in d.items()}
    loss, stats, got = check(cube)
    assert torch.equal(loss, flat[0]) and torch.equal(got[0].view(-1, v), flat[2][0]) and got[0].shape == (T, B, A, v)
    # a head's columns of a wider output, a strided batch, an int64 action
    wide = torch.randn(T * B * A, 11, device=DEV)
    wide[:, 3:8] = d["logits"].detach()
    part = dict(d, logits=wide[:, 3:8], actions=d["actions"].long(), values=d["values"].detach())
    assert torch.equal(check(part)[0], flat[0])
    wide.requires_grad_(True)
    loss, _ = mpe_hip.ppo_loss(**dict(part, logits=wide[:, 3:8]))
    (gw,) = torch.autograd.grad(loss, wide)
    assert torch.equal(gw[:, 3:8], flat[2][0]) and float(gw[:, :3].abs().sum() + gw[:, 8:].abs().sum()) == 0
    every = {k: (None if t is None else t.detach().repeat_interleave(2, 0)[::2]) for k, t in d.items()}
    assert torch.equal(check(every)[0], flat[0])
    turned = dict(d, logits=d["logits"].detach().T.contiguous().T)
    assert torch.equal(check(turned)[0], flat[0])
    half = dict(d, weights=(torch.arange(T * B * A, device=DEV) % 2 == 0))
    assert torch.equal(check(half)[0], check(dict(d, weights=half["weights"].float()))[0])


def test_upstream_gradient_scales_and_no_rows():
    import mpe_hip
    for rows, v in ((100, 5), (20, 600)):
        d = make(rows, v)
        for k in ("logits", "values"):
            d[k].requires_grad_(True)
        one = torch.autograd.grad(mpe_hip.ppo_loss(**d)[0], (d["logits"], d["values"]))
        two = torch.autograd.grad(mpe_hip.ppo_loss(**d)[0] * 1024.0, (d["logits"], d["values"]))
        assert all(torch.equal(p * 1024.0, q) for p, q in zip(one, two))
        only = torch.autograd.grad(mpe_hip.ppo_loss(**dict(d, logits=d["logits"].detach()))[0], d["values"])
        assert torch.equal(only[0], one[1])
    e = {k: (None if t is None else t.detach()[:0]) for k, t in d.items()}
    e["logits"].requires_grad_(True)
    loss, stats = mpe_hip.ppo_loss(**e)
    assert float(loss.detach()) == 0 and torch.autograd.grad(loss, e["logits"])[0].shape == (0, 600)
    loss /= 2           # a result like any other


def test_gradient_against_differences():
    """(f(+h) - f(-h)) / 2h of the kernels' own loss along a direction, h = 2^-5: off by h^2 times a third derivative (below 40
    per unit of share for these sizes, |d| <= 4) and by the loss's rounding, 64 v / h."""
    import mpe_hip
    for rows, v in ((50, 5), (20, 90), (4, 3000)):
        d = make(rows, v, values=True)
        d["old_logp"] = torch.log_softmax(d["logits"].double(), 1).gather(1, d["actions"].long()[:, None])[:, 0].float()    # ratios at 1: clear of the borders
        d["logits"].requires_grad_(True)
        (g,) = torch.autograd.grad(mpe_hip.ppo_loss(**d, entropy_coef=0.1, clip=0.5)[0], d["logits"])
        gen = torch.Generator(DEV).manual_seed(1)
        step = torch.randn(rows, v, device=DEV, generator=gen).clamp(-2, 2)
        h = 2.0 ** -5
        f = lambda s: float(mpe_hip.ppo_loss(**dict(d, logits=d["logits"].detach() + s * h * step), entropy_coef=0.1, clip=0.5)[0])
        assert abs((f(1) - f(-1)) / (2 * h) - float((g.double() * step.double()).sum())) <= 40 * h * h + 64 * V / h


def test_repeat_capture_and_streams():
    import mpe_hip
    for rows, v in ((5000, 5), (300, 70), (20, 5000)):
        d = make(rows, v, mask=True, weights=True)
        leaves = [d["logits"].requires_grad_(True), d["values"].requires_grad_(True)]
        call = lambda q: (lambda ls: [ls[0].detach(), ls[1]] + list(torch.autograd.grad(ls[0], [q["logits"], q["values"]])))(mpe_hip.ppo_loss(**q, value_clip=0.2))
        copy = lambda: {k: (None if t is None else t.detach().clone().requires_grad_(k in ("logits", "values"))) for k, t in d.items()}
        want = call(copy())
        for _ in range(2):
            assert all(torch.equal(p, q) for p, q in zip(want, call(copy())))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = call(copy())
            call(d)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(want, there))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(d)
        for i in range(3):
            with torch.no_grad():
                leaves[0].copy_(torch.randn_like(leaves[0]))
                leaves[1].copy_(torch.randn_like(leaves[1]))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, call(copy()))), (rows, v, i)
            torch.cuda.synchronize()


def test_refusals():
    import mpe_hip
    d = make(8, 5, weights=True, mask=True)
    for bad in (dict(actions=d["actions"].float()), dict(actions=d["actions"][:7]), dict(old_logp=d["old_logp"].double()), dict(advantages=d["advantages"][None]),
                dict(values=None), dict(returns=None), dict(weights=d["weights"].double()), dict(action_mask=d["action_mask"].float()),
                dict(action_mask=d["action_mask"][:, :4]), dict(logits=d["logits"].double()), dict(logits=d["logits"][:, :0]), dict(old_logp=d["old_logp"].cpu()),
                dict(clip=-0.1), dict(clip=math.nan), dict(value_clip=-0.5)):
        with pytest.raises(ValueError):
            mpe_hip.ppo_loss(**{**d, **bad})
    q = make(8, 5)
    q["logits"].requires_grad_(True)
    loss, _ = mpe_hip.ppo_loss(**q)
    q["advantages"].mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        torch.autograd.grad(loss, q["logits"])
