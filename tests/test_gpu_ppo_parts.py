"""mpe_hip.ppo_loss where only values learn, and where its inputs do not lie as rows."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def make(rows, v, dt=torch.float32):
    g = torch.Generator(DEV).manual_seed(rows + v)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)
    d = dict(logits=rnd(rows, v).to(dt), actions=torch.randint(-1, v + 1, (rows,), device=DEV, generator=g), old_logp=rnd(rows) - 1, advantages=rnd(rows), values=rnd(rows),
             old_values=rnd(rows), returns=rnd(rows), action_mask=rnd(rows, v) < 1, weights=(rnd(rows) + 0.5).clamp(min=0))
    d["logits"][::5, 0] = -float("inf")
    return d


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", [(1, 1), (75, 5), (3000, 20), (100, 300), (9, 9000)])
@pytest.mark.parametrize("value_clip", [None, 0.2])
def test_the_values_gradient_alone_has_the_same_bits(rows, v, dt, value_clip):
    import mpe_hip
    d = make(rows, v, dt)
    for mask, weights in ((True, True), (False, False)):
        q = dict(d, action_mask=d["action_mask"] if mask else None, weights=d["weights"] if weights else None)
        leaves = [q["logits"].clone().requires_grad_(True), q["values"].clone().requires_grad_(True)]
        both = torch.autograd.grad(mpe_hip.ppo_loss(**dict(q, logits=leaves[0], values=leaves[1]), value_clip=value_clip)[0], leaves)
        alone, = torch.autograd.grad(mpe_hip.ppo_loss(**dict(q, values=leaves[1]), value_clip=value_clip)[0], leaves[1:])
        assert torch.equal(alone, both[1])


def test_the_values_gradient_alone_needs_no_place_for_the_logits():
    import mpe_hip
    d = make(2000, 8192)
    values = d["values"].requires_grad_(True)
    loss, _ = mpe_hip.ppo_loss(**d)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    torch.autograd.grad(loss, values)
    assert torch.cuda.max_memory_allocated() - before < d["logits"].numel()        # a quarter of their bytes


@pytest.mark.parametrize("rows,v", [(400, 5), (300, 700)])
def test_inputs_that_are_copied_are_copied_once(rows, v):
    """Columns of a transposed tensor, a mask of one row for all: the backward pass finds the forward's copies."""
    import mpe_hip
    d = make(rows, v)
    turned = d["logits"].T.contiguous().T.requires_grad_(True)
    q = dict(d, logits=turned, action_mask=d["action_mask"][:1].expand(rows, v), values=torch.stack([d["values"]] * 2, 1)[:, 0].requires_grad_(True))
    plain = {k: t.detach().contiguous().requires_grad_(k in ("logits", "values")) for k, t in q.items()}
    loss, _ = mpe_hip.ppo_loss(**q, value_clip=0.2)
    want = torch.autograd.grad(mpe_hip.ppo_loss(**plain, value_clip=0.2)[0], [plain["logits"], plain["values"]])
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = torch.autograd.grad(loss, [turned, q["values"]], retain_graph=True)
    size = sum(t.numel() * t.element_size() for t in got)
    assert torch.cuda.max_memory_allocated() - before <= size + 2048
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[0].shape == (rows, v)
    cube = {k: t.detach().reshape((rows // 4, 4) + t.shape[1:]) for k, t in q.items()}
    cube["logits"] = turned.detach().view(rows, v).unflatten(0, (rows // 4, 4)).requires_grad_(True)
    got3, = torch.autograd.grad(mpe_hip.ppo_loss(**cube, value_clip=0.2)[0], cube["logits"])
    assert torch.equal(got3.reshape(rows, v), want[0])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,v", [(300, 31), (300, 32), (300, 33), (2000, 47), (300, 48), (259, 49), (300, 61), (1030, 62), (300, 63)])
def test_about_as_many_words_as_lanes(rows, v, dt):
    """Where a lane a row and a wave a row meet: the formula, with masks and weights."""
    from test_gpu_ppo import check
    from test_gpu_ppo import make as rollout
    check(rollout(rows, v, dt, mask=True, weights=True), value_clip=0.2)
    check(rollout(rows, v, dt, values=False))
