"""A NaN in a row of mpe_hip.ppo_loss that counts: loss and gradients show it, and nothing else does."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
ROWS, BAD = 9, 4


def make(v, seed=0):
    g = torch.Generator(DEV).manual_seed(seed + v)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
    d = dict(logits=rnd(ROWS, v), actions=torch.randint(0, v, (ROWS,), device=DEV, generator=g, dtype=torch.int32), advantages=rnd(ROWS), values=rnd(ROWS))
    d["old_logp"] = torch.log_softmax(d["logits"], 1).gather(1, d["actions"].long()[:, None])[:, 0] + 0.1
    d["old_values"], d["returns"] = d["values"] - 0.05, d["values"] + rnd(ROWS)
    return d


def run(d, **kw):
    import mpe_hip
    leaves = [d[k].requires_grad_(True) for k in ("logits", "values")]
    loss, stats = mpe_hip.ppo_loss(**d, **kw)
    dl, dv = torch.autograd.grad(loss, leaves)
    return loss.detach(), stats, dl, dv


@pytest.mark.parametrize("value_clip", [None, 0.2])
@pytest.mark.parametrize("v", [5, 20, 70, 5000])
@pytest.mark.parametrize("name", ["old_logp", "advantages", "values", "old_values", "returns", "weights", "logits"])
def test_one_nan_shows_in_the_loss_and_in_its_row(name, v, value_clip):
    good = make(v)
    want = run({k: t.clone() for k, t in good.items()}, value_clip=value_clip)
    d = make(v)
    if name == "weights":
        d["weights"] = torch.ones(ROWS, device=DEV)
    if name == "logits":
        d["logits"][BAD, (int(d["actions"][BAD]) + 1) % v] = math.nan
    else:
        d[name][BAD] = math.nan
    loss, stats, dl, dv = run(d, value_clip=value_clip)
    if name == "old_values" and value_clip is None:         # not a part of the loss then
        assert torch.equal(loss, want[0]) and torch.equal(dl, want[2]) and torch.equal(dv, want[3])
        return
    assert torch.isnan(loss)
    rest = [i for i in range(ROWS) if i != BAD]
    if name == "weights":                                   # a NaN total: every row's share
        assert torch.isnan(dl).all() and torch.isnan(dv).all() and torch.isnan(stats).all()
        return
    assert torch.equal(dl[rest], want[2][rest]) and torch.equal(dv[rest], want[3][rest])
    if name in ("values", "old_values", "returns"):
        assert torch.equal(dl[BAD], want[2][BAD]) and torch.isnan(dv[BAD]) and torch.isnan(stats[1]) and not torch.isnan(stats[0])
    else:
        assert torch.isnan(dl[BAD]).all() and torch.equal(dv[BAD], want[3][BAD]) and torch.isnan(stats[0]) and not torch.isnan(stats[1])


@pytest.mark.parametrize("v", [5, 20, 70, 5000])
def test_ratios_beyond_float32(v):
    """q = e^200: infinite in float32, a number in the formula.  Times an advantage of zero it is zero, above it the clamp holds it,
    below the loss is -infinity's opposite; q = infinity itself (an action the old policy could not take) times zero is NaN."""
    base = run(make(v))
    for adv, old, check in ((0.0, -200.0, "zero"), (2.0, -200.0, "held"), (-2.0, -200.0, "infinite"), (0.0, -math.inf, "nan"), (2.0, -math.inf, "held"), (0.0, math.inf, "zero")):
        d = make(v)
        d["advantages"][BAD], d["old_logp"][BAD] = adv, old
        loss, stats, dl, dv = run(d, entropy_coef=0.0)
        if check == "nan":
            assert torch.isnan(loss) and torch.isnan(dl[BAD]).all()
        elif check == "infinite":
            assert float(loss) == math.inf and not torch.isfinite(dl[BAD, int(d["actions"][BAD])])
        else:
            assert torch.isfinite(loss) and torch.equal(dl[BAD], torch.zeros_like(dl[BAD]))
        assert torch.equal(dv, base[3])


def test_infinite_values_follow_the_formula():
    """max((V - R)^2, (V0 + clamp(V - V0) - R)^2) / 2 in float64, element by element; a NaN in either is NaN."""
    import itertools
    import mpe_hip
    nums = [0.0, 1.5, math.inf, -math.inf, math.nan]
    for V, V0, R in itertools.product(nums, nums, nums):
        t = lambda x: torch.tensor([x], device=DEV)
        vals = t(V).requires_grad_(True)
        loss, stats = mpe_hip.ppo_loss(torch.zeros(1, 2, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), t(-0.69), t(0.0), vals, t(V0), t(R), value_clip=0.2)
        a, b, c = (torch.tensor(x, dtype=torch.float64) for x in (V, V0, R))
        want = torch.maximum((a - c) ** 2, (b + (a - b).clamp(-torch.tensor(0.2).double(), torch.tensor(0.2).double()) - c) ** 2) / 2
        got = float(stats[1])
        assert math.isnan(got) if math.isnan(float(want)) else got == float(want) or abs(got - float(want)) <= 2.0 ** -22 * abs(float(want)), (V, V0, R, got, float(want))


def test_every_negative_value_clip_is_refused():
    """Also the number that stands for "not clipped" behind the C boundary."""
    import mpe_hip
    d = make(5)
    for bad in (-1.0, -1, -0.5, -1e-60, math.nan):
        with pytest.raises(ValueError, match="value_clip"):
            mpe_hip.ppo_loss(**d, value_clip=bad)
    assert torch.equal(mpe_hip.ppo_loss(**d, value_clip=math.inf)[0], mpe_hip.ppo_loss(**d)[0])


def test_a_value_clip_below_zero_by_less_than_float32_holds_does_not_clip():
    """Behind the C boundary, where every negative value_clip means none."""
    from mpe_hip import _lib
    lib, d = _lib.load(), make(5)
    def stats(value_clip):
        loss, out, ws = torch.empty(1, device=DEV), torch.empty(6, device=DEV), torch.empty(_lib.PPO_WORKSPACE_BYTES, dtype=torch.uint8, device=DEV)
        p = {k: t.contiguous().data_ptr() for k, t in d.items()}
        assert lib.mpe_ppo_loss_forward(0, _lib.MPE_F32, ROWS, 5, p["logits"], 5, p["actions"], 4, p["old_logp"], p["advantages"], None, 0, None, p["values"], p["old_values"],
                                        p["returns"], 0.2, value_clip, 0.5, 0.01, loss.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(),
                                        torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        return out
    assert torch.equal(stats(-1e-60), stats(-1.0)) and not torch.equal(stats(0.0), stats(-1.0))
