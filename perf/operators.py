"""The trainer-side operators that are measured: a policy's layers, its loss and the clipping of its gradients.

What a training loop runs between two rollouts of the batched worlds: ``linear`` (product, bias, activation and
residual) over the observations of all agents, ``ppo_loss`` (clipped surrogate, value loss and entropy, with the
gradient) over the rollout that ``gae`` gave advantages to, and the clipping of the gradients to a global norm.

``listed()`` gives the fixed cases, ``draw(rng)`` further ones of the same ranges, ``prepare`` a case's inputs,
``run`` one pass (with ``own`` the framework's calls, without it the plain torch form), ``exact`` the same outputs from
the definitions in 64 bits, ``work`` the bytes and operations that a pass cannot do without.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_MAX_FLOPS = 3 * 2 * 65536 * 1024 * 1024        # the largest listed case's operations
_MAX_CLIP = 24 * 12 * 1024 * 1024               # elements of the largest listed list of gradients
_MAX_LOGITS = 25 * 65536 * 3 * 5 * 4 // 3       # logits of the largest loss, about


def listed():
    return [
        # one simple_spread world acting: 3 agents' 14-wide observations through the policy's first layer
        {"name": "act_one_world", "op": "linear", "m": 3, "k": 14, "n": 64, "ld": 14, "dtype": "f32", "act": "tanh", "bias": True, "residual": False},
        # one agent's layer for the headline batch: its columns of the [65536, 42] observations, row stride 42
        {"name": "act_agent_view", "op": "linear", "m": 65536, "k": 14, "n": 64, "ld": 42, "dtype": "f32", "act": "tanh", "bias": True, "residual": False},
        # 64-agent worlds, 2048 of them: the 258-wide observations of every agent into a wide first layer
        {"name": "act_wide", "op": "linear", "m": 131072, "k": 258, "n": 512, "ld": 258, "dtype": "bf16", "act": "silu", "bias": True, "residual": False},
        # one decision of one world through a wide trunk: the weights are the traffic
        {"name": "act_trunk_token", "op": "linear", "m": 4, "k": 1024, "n": 4096, "ld": 1024, "dtype": "bf16", "act": "gelu", "bias": True, "residual": False},
        # a hidden layer of the usual small policy, update over one step of all agents of the headline batch
        {"name": "learn_hidden", "op": "learn", "m": 196608, "k": 64, "n": 64, "ld": 64, "dtype": "f32", "act": "tanh", "bias": True, "residual": False, "dx": True},
        # a ragged minibatch through a layer with odd sizes and a skip connection
        {"name": "learn_ragged", "op": "learn", "m": 10007, "k": 258, "n": 255, "ld": 258, "dtype": "f32", "act": "gelu", "bias": True, "residual": True, "dx": True},
        # one block of a wide residual trunk over a large minibatch
        {"name": "learn_block", "op": "learn", "m": 65536, "k": 1024, "n": 1024, "ld": 1024, "dtype": "bf16", "act": "gelu", "bias": True, "residual": True, "dx": True},
        # gradients of a two-layer policy and value net of width 64
        {"name": "clip_policy", "op": "clip", "kind": "policy", "width": 64, "layers": 2, "dtype": "f32", "max_norm": 0.5, "spread": 1.0},
        # gradients of a 24-layer trunk of width 1024 in bfloat16, its vectors in float32
        {"name": "clip_trunk", "op": "clip", "kind": "trunk", "width": 1024, "layers": 24, "dtype": "bf16", "max_norm": 1.0, "spread": 0.01},
        # the smallest update: one episode of one world, 25 steps of 3 agents
        {"name": "loss_one_world", "op": "loss", "rows": 75, "v": 5, "dtype": "f32", "values": True, "mask": False, "weights": False, "scale": 1.0},
        # a whole rollout of the headline batch: 25 steps x 65536 worlds x 3 agents, 5 moves
        {"name": "loss_rollout", "op": "loss", "rows": 25 * 65536 * 3, "v": 5, "dtype": "f32", "values": True, "mask": False, "weights": False, "scale": 1.0},
        # agents that answer with words: a large vocabulary, disallowed words masked, padded steps
        {"name": "loss_words", "op": "loss", "rows": 4096, "v": 8192, "dtype": "bf16", "values": False, "mask": True, "weights": True, "scale": 1.0},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _rough(rng, n, lo):
    """n as drawn, or the nearest multiple of 64: real layers have both."""
    return n if rng.random() < 0.5 else max(lo, (n + 32) // 64 * 64)


def draw(rng):
    op = rng.choice(["linear", "linear", "learn", "learn", "clip", "loss", "loss"])
    if op in ("linear", "learn"):
        m = _log_int(rng, 1 if op == "linear" else 64, 196608)
        k = _rough(rng, _log_int(rng, 3, 1024), 3)
        n = _rough(rng, _log_int(rng, 1, 4096 if op == "linear" else 1024), 1)
        passes = 1 if op == "linear" else 3
        m = max(1, min(m, _MAX_FLOPS // (passes * 2 * k * n)))
        # a row stride beyond the width: one agent's columns of a row that holds several agents'
        ld = k * rng.choice([2, 3]) if rng.random() < 0.25 else k
        act = rng.choice(["tanh", "gelu", "silu", "relu", "none"] if op == "linear" else ["tanh", "gelu", "silu", "none"])
        case = {"op": op, "m": m, "k": k, "n": n, "ld": ld, "dtype": rng.choice(["f32", "bf16", "f16"]), "act": act,
                "bias": rng.random() < 0.8, "residual": rng.random() < 0.3}
        if op == "learn":
            case["dx"] = rng.random() < 0.7
        return case
    if op == "clip":
        kind = rng.choice(["policy", "trunk", "odd"])
        layers = rng.randint(1, 24)
        width = _log_int(rng, 16, 1024)
        while _clip_count(kind, width, layers) > _MAX_CLIP:
            layers -= 1
        return {"op": "clip", "kind": kind, "width": width, "layers": layers, "dtype": rng.choice(["f32", "bf16", "f16"]),
                "max_norm": rng.choice([0.5, 1.0, 10.0]), "spread": rng.choice([1e-4, 0.01, 1.0])}
    dtype = rng.choice(["f32", "bf16", "f16"])
    v = _log_int(rng, 2, 8192)
    rows = _log_int(rng, 1, 4000000)
    rows = max(1, min(rows, _MAX_LOGITS // v, 4915200))
    return {"op": "loss", "rows": rows, "v": v, "dtype": dtype, "values": rng.random() < 0.5, "mask": rng.random() < 0.4,
            "weights": rng.random() < 0.4, "scale": 1.0 if dtype != "f16" else float(2 ** max(0, math.ceil(math.log2(rows))))}


# ---- inputs ---------------------------------------------------------------------------------------------------------

def _shapes(kind, width, layers):
    """(shape, is a vector) of every gradient of a model."""
    out = []
    if kind == "policy":        # observation -> hidden layers -> 5 moves, and the same again for the value
        for head in (5, 1):
            k = 14
            for _ in range(layers):
                out += [((width, k), False), ((width,), True)]
                k = width
            out += [((head, k), False), ((head,), True)]
    elif kind == "trunk":       # per layer: the four square matrices of an attention and two of a four times wider product
        for _ in range(layers):
            out += [((width, width), False)] * 4 + [((4 * width, width), False), ((width, 4 * width), False)]
            out += [((width,), True)] * 4
    else:                       # odd lengths, one-element tensors
        for i in range(layers):
            out += [((width + i, 2 * i + 3), False), ((1,), True), ((width * 7 + 3 * i + 1,), True)]
    return out


def _types(grads):
    return sorted({t.dtype for t in grads}, key=str)


def _clip_count(kind, width, layers):
    return sum(math.prod(s) for s, _ in _shapes(kind, width, layers))


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _framework():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "multiagent-particle-envs_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import mpe_hip
    return mpe_hip


def prepare(case, seed):
    g = _gen(seed)
    dev = "cuda"
    op, dt = case["op"], _DTYPES[case["dtype"]]
    st = {"case": case}
    normal = lambda *s: torch.randn(*s, device=dev, generator=g)
    if op in ("linear", "learn"):
        m, k, n, ld = case["m"], case["k"], case["n"], case["ld"]
        st["x"] = normal(m, ld).to(dt)[:, ld - k:]
        st["w"] = (normal(n, k) / math.sqrt(k)).to(dt)
        st["b"] = (0.1 * normal(n)).to(dt) if case["bias"] else None
        st["r"] = normal(m, n).to(dt) if case["residual"] else None
        if op == "learn":
            st["dy"] = (0.1 * normal(m, n)).to(dt)
            st["leaves"] = [t for t, need in ((st["x"], case["dx"]), (st["w"], True), (st["b"], True), (st["r"], True)) if need and t is not None]
            if own:
                for t in st["leaves"]:
                    t.requires_grad_(True)
    elif op == "clip":
        st["grads"] = [(case["spread"] * normal(*s)).to(torch.float32 if vec else dt) for s, vec in _shapes(case["kind"], case["width"], case["layers"])]
        # the optimiser reads flat buffers, one a type; every clipped gradient is a slice of its type's
        st["flat"] = [torch.empty(sum(t.numel() for t in st["grads"] if t.dtype == d), dtype=d, device=dev) for d in _types(st["grads"])]
        st["out"], at = [], {f.dtype: 0 for f in st["flat"]}
        for t in st["grads"]:
            flat = st["flat"][_types(st["grads"]).index(t.dtype)]
            st["out"].append(flat[at[t.dtype]:at[t.dtype] + t.numel()].view(t.shape))
            at[t.dtype] += t.numel()
    else:
        r, v = case["rows"], case["v"]
        logits = (1.5 * normal(r, v)).to(dt)
        rand = lambda *s: torch.rand(*s, device=dev, generator=g)
        allowed = None
        if case["mask"]:
            allowed = rand(r, v) < 0.7
            allowed[5::97] = False              # an agent with no word left
        # the action was drawn by the policy that collected the rollout
        score = logits.float() - torch.log(-torch.log(rand(r, v).clamp(1e-7, 1 - 1e-7)))
        if allowed is not None:
            score = score.masked_fill(~allowed, -1e30)
        act = score.argmax(1)
        del score
        # that policy was a little different: its log-probability is the present one less a log-ratio that stays clear of
        # the clipping borders by 1e-3, where the last bit of an exponential would decide the branch
        log_ratio = 0.15 * normal(r).double()
        ratio = log_ratio.exp()
        for border in (0.8, 1.2):
            near = (ratio - border).abs() < 1e-3
            log_ratio = torch.where(near, torch.full_like(log_ratio, math.log(border + 2e-3)), log_ratio)
            ratio = log_ratio.exp()
        old = torch.empty(r, device=dev)
        for i in range(0, r, 1 << 20):          # in pieces: 64-bit logits of a whole rollout are large
            l64 = logits[i:i + (1 << 20)].double()
            if allowed is not None:
                l64 = l64.masked_fill(~allowed[i:i + (1 << 20)], -math.inf)
            lp = l64.gather(1, act[i:i + (1 << 20), None])[:, 0] - torch.logsumexp(l64, 1)
            old[i:i + (1 << 20)] = torch.where(torch.isfinite(lp), lp - log_ratio[i:i + (1 << 20)], torch.zeros_like(lp)).float()
        st.update(logits=logits, actions=act.to(torch.int32), old_logp=old, adv=normal(r), allowed=allowed)
        st["weights"] = None
        if case["weights"]:
            st["weights"] = (rand(r) < 0.9).float()
            st["weights"][r - r // 8:] = 0.0    # steps behind the end of the episodes
        st["values"] = st["old_values"] = st["returns"] = None
        if case["values"]:
            st["old_values"] = normal(r)
            st["values"] = st["old_values"] + 0.2 * normal(r)
            st["returns"] = st["old_values"] + normal(r)
        st["grad"] = torch.full((), case["scale"], device=dev)
        if own:
            st["leaves"] = [t for t in (st["logits"], st["values"]) if t is not None]
            for t in st["leaves"]:
                t.requires_grad_(True)
    if own:
        st["mpe"] = _framework()
    return st


_CLIP, _VCLIP, _VCOEF, _ECOEF = 0.2, 0.2, 0.5, 0.01


# ---- one pass -------------------------------------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if own:
        mpe, case = st["mpe"], st["case"]
        if op == "linear":
            return mpe.linear(st["x"], st["w"], st["b"], activation=case["act"], residual=st["r"])
        if op == "learn":
            y = mpe.linear(st["x"], st["w"], st["b"], activation=case["act"], residual=st["r"])
            return [y.detach()] + list(torch.autograd.grad(y, st["leaves"], st["dy"]))
        if op == "clip":
            norm = mpe.clip_grad_norm(st["grads"], case["max_norm"], out=st["out"])
            return [norm] + st["flat"]
        loss, stats = mpe.ppo_loss(st["logits"], st["actions"], st["old_logp"], st["adv"], values=st["values"], old_values=st["old_values"],
                                   returns=st["returns"], action_mask=st["allowed"], weights=st["weights"], clip=_CLIP, value_clip=_VCLIP,
                                   value_coef=_VCOEF, entropy_coef=_ECOEF)
        return [loss.detach(), stats] + list(torch.autograd.grad(loss, st["leaves"], st["grad"]))
    return {"linear": _plain_linear, "learn": _plain_learn, "clip": _plain_clip, "loss": _plain_loss}[op](st)


_INV_SQRT2, _INV_SQRT2PI = 1.0 / math.sqrt(2.0), 1.0 / math.sqrt(2.0 * math.pi)


def _plain_act(z, act):
    if act == "tanh":
        return torch.tanh(z)
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * _INV_SQRT2))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _plain_slope(z, act):
    if act == "tanh":
        t = torch.tanh(z)
        return 1 - t * t
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * _INV_SQRT2)) + z * _INV_SQRT2PI * torch.exp(-0.5 * z * z)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain_pre(st):
    z = torch.matmul(st["x"].float(), st["w"].float().t())
    return z if st["b"] is None else z + st["b"].float()


def _plain_linear(st):
    y = _plain_act(_plain_pre(st), st["case"]["act"])
    if st["r"] is not None:
        y = y + st["r"].float()
    return y.to(st["x"].dtype)


def _plain_learn(st):
    case, dt = st["case"], st["x"].dtype
    z = _plain_pre(st)
    y = _plain_act(z, case["act"])
    if st["r"] is not None:
        y = y + st["r"].float()
    dy = st["dy"].float()
    dz = dy * _plain_slope(z, case["act"])
    out = [y.to(dt)]
    if case["dx"]:
        out.append(torch.matmul(dz, st["w"].float()).to(dt))
    out.append(torch.matmul(dz.t(), st["x"].float()).to(dt))
    if st["b"] is not None:
        out.append(dz.sum(0).to(dt))
    if st["r"] is not None:
        out.append(st["dy"].clone())
    return out


def _plain_clip(st):
    total = torch.stack([(t.double() * t.double()).sum() for t in st["grads"]]).sum()
    norm = torch.sqrt(total)
    scale = (st["case"]["max_norm"] / torch.clamp(norm, min=st["case"]["max_norm"])).float()
    for t, out in zip(st["grads"], st["out"]):
        out.copy_((t.float() * scale).to(t.dtype))
    return [norm.float()] + st["flat"]


def _plain_loss(st):
    l = st["logits"].float()
    r, v = l.shape
    live = torch.ones(r, device=l.device) if st["weights"] is None else st["weights"]
    if st["allowed"] is not None:
        some = st["allowed"].any(1)
        live = live * some
        l = torch.where(st["allowed"] | ~some[:, None], l, torch.full_like(l, -1e30))
    e = torch.exp(l - l.amax(1, keepdim=True))
    s = e.sum(1, keepdim=True)
    p = e / s
    logp = l - l.amax(1, keepdim=True) - torch.log(s)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    ent = -plogp.sum(1)
    at = logp.gather(1, st["actions"].long()[:, None])[:, 0]
    diff = at - st["old_logp"]
    ratio = torch.exp(diff)
    adv = st["adv"]
    held = torch.clamp(ratio, 1 - _CLIP, 1 + _CLIP)
    moves = ratio * adv <= held * adv
    pg = -torch.minimum(ratio * adv, held * adv)
    total = live.double().sum()
    total = torch.where(total > 0, total, torch.ones_like(total))       # no live row: nothing to learn, loss 0
    mean = lambda t: ((t.double() * live.double()).sum() / total)
    zero = torch.zeros((), dtype=torch.float64, device=l.device)
    policy, entropy = mean(pg), mean(ent)
    value = zero
    share = (st["grad"].double() * live.double() / total).float()
    out = []
    if st["values"] is not None:
        val, old, ret = st["values"].double(), st["old_values"].double(), st["returns"].double()
        step = val - old
        free, tied = val - ret, old + torch.clamp(step, -_VCLIP, _VCLIP) - ret
        value = mean(0.5 * torch.maximum(free * free, tied * tied))
        slope = torch.where(free * free >= tied * tied, free, torch.where(step.abs() <= _VCLIP, tied, torch.zeros_like(tied)))
        out = [(share.double() * _VCOEF * slope).float()]
    stats = torch.stack([policy, value, entropy, mean(0.5 * diff * diff), mean(((ratio - 1).abs() > _CLIP).float())])
    loss = policy + _VCOEF * value - _ECOEF * entropy
    c1 = torch.where(moves, -ratio * adv, torch.zeros_like(adv)) * share
    c2 = _ECOEF * share
    dl = -c1[:, None] * p + c2[:, None] * (plogp + p * ent[:, None])
    dl.scatter_add_(1, st["actions"].long()[:, None], c1[:, None])
    return [loss.float(), stats.float(), dl.to(st["logits"].dtype)] + out


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    """The definitions in float64; gradients by differentiating the scalar <outputs, upstream gradient> itself."""
    st = prepare(case, seed)
    f64 = lambda t: None if t is None else t.detach().to(torch.float64)
    if case["op"] == "clip":
        sq = 0.0
        for t in st["grads"]:
            sq = sq + f64(t).pow(2).sum()
        norm = sq.sqrt()
        factor = case["max_norm"] / norm if norm > case["max_norm"] else 1.0
        return [norm] + [torch.cat([f64(t).flatten() * factor for t in st["grads"] if t.dtype == d]) for d in _types(st["grads"])]
    if case["op"] in ("linear", "learn"):
        leaves = {k: f64(st[k]) for k in ("x", "w", "b", "r") if st[k] is not None}
        learn = case["op"] == "learn"
        if learn:
            for k, t in leaves.items():
                t.requires_grad_(k != "x" or case["dx"])
        with torch.set_grad_enabled(learn):
            z = leaves["x"] @ leaves["w"].T
            if "b" in leaves:
                z = z + leaves["b"]
            if case["act"] == "tanh":
                a = z.tanh()
            elif case["act"] == "relu":
                a = z * (z > 0)
            elif case["act"] == "gelu":
                a = z * (0.5 * torch.erfc(-z / math.sqrt(2.0)))
            elif case["act"] == "silu":
                a = z * torch.sigmoid(z)
            else:
                a = z * 1.0
            y = a + leaves["r"] if "r" in leaves else a
        if not learn:
            return y
        wanted = [t for t in leaves.values() if t.requires_grad]
        return [y.detach()] + list(torch.autograd.grad(y, wanted, f64(st["dy"])))
    rows = st["logits"].shape[0]
    logits = f64(st["logits"]).requires_grad_(True)
    values = f64(st["values"])
    w = torch.ones(rows, dtype=torch.float64, device=logits.device) if st["weights"] is None else f64(st["weights"])
    with torch.enable_grad():
        scores = logits
        if st["allowed"] is not None:
            empty = ~st["allowed"].any(dim=-1)
            w = w.masked_fill(empty, 0.0)
            scores = logits.masked_fill(~(st["allowed"] | empty[:, None]), -1e300)
        logp = scores.log_softmax(-1)
        ent = -(logp.exp() * logp.clamp(min=-1e4)).sum(-1)
        diff = logp[torch.arange(rows, device=logits.device), st["actions"].long()] - f64(st["old_logp"])
        ratio, adv = diff.clamp(max=500.0).exp(), f64(st["adv"])
        surrogate = torch.min(ratio * adv, ratio.clamp(1 - _CLIP, 1 + _CLIP) * adv)
        share = w / w.sum() if w.any() else w
        policy, entropy = -(share * surrogate).sum(), (share * ent).sum()
        value = torch.zeros((), dtype=torch.float64, device=logits.device)
        if values is not None:
            values.requires_grad_(True)
            old, ret = f64(st["old_values"]), f64(st["returns"])
            near = old + (values - old).clamp(-_VCLIP, _VCLIP)
            value = 0.5 * (share * torch.max((values - ret) ** 2, (near - ret) ** 2)).sum()
        loss = policy + _VCOEF * value - _ECOEF * entropy
    stats = torch.stack([policy, value, entropy, (share * diff ** 2).sum() / 2, (share * ((ratio > 1 + _CLIP) | (ratio < 1 - _CLIP))).sum()]).detach()
    wanted = [logits] + ([values] if values is not None else [])
    return [loss.detach(), stats] + list(torch.autograd.grad(loss, wanted, f64(st["grad"])))


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    s = _SIZE[case["dtype"]]
    if case["op"] in ("linear", "learn"):
        m, k, n = case["m"], case["k"], case["n"]
        xs, ws, ys = m * k * s, n * k * s, m * n * s
        b = n * s if case["bias"] else 0
        res = ys if case["residual"] else 0
        if case["op"] == "linear":
            return {"bytes": xs + ws + b + res + ys, "flops": 2 * m * k * n}
        # forward as above; dy read, the gradients written (the residual's is dy itself)
        return {"bytes": xs + ws + b + res + ys + ys + ws + b + (xs if case["dx"] else 0), "flops": (6 if case["dx"] else 4) * m * k * n}
    if case["op"] == "clip":
        shapes = _shapes(case["kind"], case["width"], case["layers"])
        size = sum(math.prod(sh) * (4 if vec else s) for sh, vec in shapes)
        return {"bytes": 2 * size + 4, "flops": 3 * _clip_count(case["kind"], case["width"], case["layers"])}
    r, v = case["rows"], case["v"]
    size = 2 * r * v * s + (r * v if case["mask"] else 0) + r * 12 + (4 * r if case["weights"] else 0) + (16 * r if case["values"] else 0) + 24
    return {"bytes": size, "flops": 12 * r * v}
