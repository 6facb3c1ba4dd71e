"""Trainer-side operators: what the policy update runs on a rollout that :func:`mpe_hip.gae` gave advantages to.

* ``linear``: a layer, ``f(x W^T + b) + r`` in one launch, with its gradients;
* ``ppo_loss``: the clipped policy loss with value loss and entropy bonus, with its gradients;
* ``clip_grad_norm`` / ``clip_grad_norm_`` / ``grad_norm``: the global norm over many tensors, and clipping to it.

All take GPU tensors (float32, bfloat16 or float16; there is no CPU path), enqueue on the current stream of the tensors'
device and return without synchronising.  All may be captured into a graph; a backward pass that is captured follows
autograd's own rule that no eager graph of the same leaves is alive.  Second derivatives are not available.
"""
import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.MPE_F32, torch.bfloat16: _lib.MPE_BF16, torch.float16: _lib.MPE_F16}
ACTIVATIONS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "tanh": _lib.ACT_TANH, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
               "silu": _lib.ACT_SILU}


_ROW_MAX = 1 << 22      # the longest row stride the kernels take


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _check(code):
    if code != 0:
        _lib.check(None, code)


def _dtype(t, what):
    if t.device.type != "cuda":
        raise ValueError("%s needs GPU tensors; there is no CPU path" % what)
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise ValueError("%s takes float32, bfloat16 or float16, not %s" % (what, t.dtype)) from None


def _rows(t, cols):
    """``t`` as a matrix of ``cols`` columns whose rows are contiguous (any row stride >= cols), copied only if it has to be."""
    m = t if t.dim() == 2 else t.reshape(-1, cols)
    if cols > 1 and m.stride(1) != 1 or (m.shape[0] > 1 and not cols <= m.stride(0) <= _ROW_MAX):
        m = m.contiguous()
    return m


def _ld(m):
    """Row stride of what _rows returned; a single row's stride says nothing."""
    return m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _rows_or_one(t, cols):
    """As _rows, but one row repeated by ``expand`` stays one row (stride 0)."""
    if t.dim() >= 2 and t.numel() > 0 and (cols == 1 or t.stride(-1) == 1) and all(s == 0 or n == 1 for s, n in zip(t.stride()[:-1], t.shape[:-1])):
        return t.as_strided((t.numel() // cols, cols), (0, 1)), 0
    m = _rows(t, cols)
    return m, _ld(m)


# ---- linear -------------------------------------------------------------------------------------------------------------

_ws_bytes = {}


def _workspace(dtype, act, m, n, k):
    key = (dtype, act, m, n, k)
    got = _ws_bytes.get(key)
    if got is None:
        f, b = C.c_int64(), C.c_int64()
        _check(_lib.load().mpe_linear_workspace(dtype, act, m, n, k, C.byref(f), C.byref(b)))
        if len(_ws_bytes) >= 4096:
            _ws_bytes.clear()
        got = _ws_bytes[key] = (f.value, b.value)
    return got


def _space(nbytes, device):
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _linear_forward(x, weight, bias, residual, act, code, keep_pre):
    n, k = weight.shape
    x2, w2 = _rows(x, k), _rows(weight, k)
    m = x2.shape[0]
    dev = x.device
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
    pre = torch.empty(m, n, dtype=x.dtype if act == _lib.ACT_RELU else torch.float32, device=dev) if keep_pre else None
    r2, ldr = (None, 0) if residual is None else _rows_or_one(residual, n)
    b1 = None if bias is None else bias.contiguous()
    ws_bytes = _workspace(code, act, m, n, k)[0]
    ws = _space(ws_bytes, dev)
    _check(_lib.load().mpe_linear_forward(dev.index, code, act, m, n, k, x2.data_ptr(), _ld(x2), w2.data_ptr(), _ld(w2), _ptr(b1), _ptr(r2), ldr,
                                          y.data_ptr(), n, _ptr(pre), _ptr(ws), ws_bytes, _stream(dev)))
    return y, pre


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, code):
        # where nothing was added to it, the output itself tells relu's slope, and in float32 tanh's
        from_y = residual is None and (act == _lib.ACT_RELU or (act == _lib.ACT_TANH and code == _lib.MPE_F32))
        own_pre = act != _lib.ACT_NONE and not from_y
        y, pre = _linear_forward(x, weight, bias, residual, act, code, own_pre)
        if from_y and act == _lib.ACT_TANH:
            act = _lib.ACT_TANH_OUT
        ctx.act, ctx.code, ctx.has_bias = act, code, bias is not None
        ctx.save_for_backward(x, weight, pre if own_pre else y if act != _lib.ACT_NONE else None)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        need_b = need_b and ctx.has_bias
        dx = dw = db = None
        if need_x or need_w or need_b:
            n, k = weight.shape
            x2, w2 = _rows(x, k), _rows(weight, k)
            m = x2.shape[0]
            dev = x.device
            dy2, lddy = _rows_or_one(dy, n)
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
            dw = torch.empty(n, k, dtype=x.dtype, device=dev) if need_w else None
            db = torch.empty(n, dtype=x.dtype, device=dev) if need_b else None
            ws_bytes = _workspace(ctx.code, ctx.act, m, n, k)[1]
            ws = _space(ws_bytes, dev)
            _check(_lib.load().mpe_linear_backward(dev.index, ctx.code, ctx.act, m, n, k, _ptr(dy2), lddy, x2.data_ptr(), _ld(x2), w2.data_ptr(),
                                                   _ld(w2), _ptr(pre), _ptr(dx), k, _ptr(dw), _ptr(db), _ptr(ws), ws_bytes, _stream(dev)))
        return dx, dw, db, dy if need_r else None, None, None


def linear(x, weight, bias=None, activation=None, residual=None):
    """``activation(x @ weight.T + bias) + residual`` in one launch, differentiable in all four.

    ``x`` ``[..., k]`` (rows may be strided: ``env.obs_n[i]`` is taken as it lies), ``weight`` ``[n, k]``, ``bias`` ``[n]``,
    ``residual`` of the result's shape ``[..., n]`` (an expanded tensor will do); all of one type (float32, bfloat16,
    float16) on one GPU.  ``activation``: None / "none", "tanh", "relu", "gelu" (by erf) or "silu".  Sums are in float32 or
    better, with one rounding to the type at the end; float32 products are as exact as float32 multiplications.  For the
    backward pass the pre-activations are kept in float32 (nothing is kept for none, relu and float32 tanh without residual)."""
    try:
        act = ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError("linear: activation must be one of none, tanh, relu, gelu, silu; got %r" % (activation,)) from None
    code = _dtype(x, "linear")
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("linear: x [..., k] and weight [n, k], n and k at least 1; got %s and %s" % (tuple(x.shape), tuple(weight.shape)))
    n = weight.shape[0]
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError("linear: bias must have shape (%d,), got %s" % (n, tuple(bias.shape)))
    if residual is not None and residual.shape != x.shape[:-1] + (n,):
        raise ValueError("linear: residual must have the result's shape %s, got %s" % (tuple(x.shape[:-1]) + (n,), tuple(residual.shape)))
    for t in (weight, bias, residual):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError("linear: all tensors must share x's type and device (%s, %s)" % (x.dtype, x.device))
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act, code)
    return _linear_forward(x, weight, bias, residual, act, code, False)[0]


# ---- ppo_loss -------------------------------------------------------------------------------------------------------------

class _PpoLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, shared, coefs, code):
        actions, old_logp, adv, old_values, returns, mask, weights = shared
        v = logits.shape[-1]
        l2 = _rows(logits, v)
        dev = logits.device
        loss, stats = torch.empty((), dtype=torch.float32, device=dev), torch.empty(6, dtype=torch.float32, device=dev)
        ws = _space(_lib.PPO_WORKSPACE_BYTES, dev)
        val = None if values is None else values.contiguous()
        args = (dev.index, code, l2.shape[0], v, l2.data_ptr(), _ld(l2), actions.data_ptr(), actions.element_size(), old_logp.data_ptr(), adv.data_ptr(),
                _ptr(mask), 0 if mask is None else _ld(mask), _ptr(weights), _ptr(val), _ptr(old_values), _ptr(returns)) + coefs
        _check(_lib.load().mpe_ppo_loss_forward(*args, loss.data_ptr(), stats.data_ptr(), ws.data_ptr(), _lib.PPO_WORKSPACE_BYTES, _stream(dev)))
        ctx.args, ctx.values_shape = args, None if values is None else values.shape
        ctx.save_for_backward(logits, values, stats, *shared)
        ctx.kept = (l2, val)        # what args point to, where it is a copy
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        logits, values, stats = ctx.saved_tensors[:3]       # raises where an input was written since
        need_l, need_v = ctx.needs_input_grad[0], ctx.needs_input_grad[1] and values is not None
        if not (need_l or need_v):
            return None, None, None, None, None
        dev = logits.device
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
        dvalues = torch.empty(ctx.values_shape, dtype=torch.float32, device=dev) if need_v else None
        grad = grad.to(torch.float32)
        _check(_lib.load().mpe_ppo_loss_backward(*ctx.args, stats.data_ptr(), grad.data_ptr(), dlogits.data_ptr(), logits.shape[-1], _ptr(dvalues), _stream(dev)))
        return dlogits if need_l else None, dvalues, None, None, None


def ppo_loss(logits, actions, old_logp, advantages, values=None, old_values=None, returns=None, action_mask=None, weights=None, clip=0.2,
             value_clip=None, value_coef=0.5, entropy_coef=0.01):
    """The clipped policy loss of a rollout, differentiable in ``logits`` and ``values``.

    ``logits`` ``[..., v]`` (float32, bfloat16, float16; rows may be strided); everything else has its leading shape:
    ``actions`` int32 / int64, ``old_logp`` and ``advantages`` float32, optionally ``values``, ``old_values`` and
    ``returns`` float32 (together), ``action_mask`` bool / uint8 ``[..., v]`` (0 forbids a move) and ``weights`` float32 /
    bool.  Per decision, with the softmax over the allowed moves: ``q = exp(logp - old_logp)``,
    ``s = min(q A, clamp(q, 1 - clip, 1 + clip) A)``, the entropy ``H`` and the value loss
    ``u = max((V - R)^2, (V0 + clamp(V - V0, -value_clip, value_clip) - R)^2) / 2`` (``value_clip`` None: ``(V - R)^2 / 2``);
    ``loss = sum w (-s + value_coef u - entropy_coef H) / sum w``.

    A decision is left out, with zero gradients, if its weight is 0 or its action lies outside ``[0, v)``, is forbidden or
    has the logit -infinity (so also where no move is left).  Returns ``(loss, stats)``: a float32 scalar and the float32 means
    ``[-s, u, H, (logp - old_logp)^2 / 2, share of clipped decisions]``."""
    code = _dtype(logits, "ppo_loss")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("ppo_loss: logits must be [..., v] with v at least 1, got %s" % (tuple(logits.shape),))
    lead, dev = logits.shape[:-1], logits.device
    if (values is None) != (old_values is None) or (values is None) != (returns is None):
        raise ValueError("ppo_loss: values, old_values and returns go together")
    if actions.dtype not in (torch.int32, torch.int64):
        raise ValueError("ppo_loss: actions must be int32 or int64, not %s" % actions.dtype)
    for name, t, want in (("old_logp", old_logp, torch.float32), ("advantages", advantages, torch.float32), ("values", values, torch.float32),
                          ("old_values", old_values, torch.float32), ("returns", returns, torch.float32)):
        if t is not None and t.dtype != want:
            raise ValueError("ppo_loss: %s must be float32, not %s" % (name, t.dtype))
    if weights is not None and weights.dtype == torch.bool:
        weights = weights.float()
    if weights is not None and weights.dtype != torch.float32:
        raise ValueError("ppo_loss: weights must be float32 or bool, not %s" % weights.dtype)
    if action_mask is not None and action_mask.dtype not in (torch.bool, torch.uint8):
        raise ValueError("ppo_loss: action_mask must be bool or uint8, not %s" % action_mask.dtype)
    for name, t, shape in (("actions", actions, lead), ("old_logp", old_logp, lead), ("advantages", advantages, lead), ("values", values, lead),
                           ("old_values", old_values, lead), ("returns", returns, lead), ("weights", weights, lead), ("action_mask", action_mask, logits.shape)):
        if t is not None and (t.shape != shape or t.device != dev):
            raise ValueError("ppo_loss: %s must have shape %s on %s, got %s on %s" % (name, tuple(shape), dev, tuple(t.shape), t.device))
    clip, value_clip = float(clip), -1.0 if value_clip is None else float(value_clip)
    if not clip >= 0 or not (value_clip >= 0 or value_clip == -1.0):
        raise ValueError("ppo_loss: clip and value_clip must not be negative")
    flat = lambda t: None if t is None else t.detach().contiguous()
    shared = (flat(actions), flat(old_logp), flat(advantages), flat(old_values), flat(returns),
              None if action_mask is None else _rows(action_mask, logits.shape[-1]), flat(weights))
    loss, stats = _PpoLoss.apply(logits, values, shared, (clip, value_clip, float(value_coef), float(entropy_coef)), code)
    return loss, stats[:5]


# ---- global norm -------------------------------------------------------------------------------------------------------------

def _dense(t):
    """True if t's elements fill one run of memory, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if s != want:
            return False
        want *= n
    return True


def _clip(tensors, max_norm, outs):
    n = len(tensors)
    dev = tensors[0].device
    src, cnt, typ = (C.c_void_p * n)(), (C.c_int64 * n)(), (C.c_int32 * n)()
    for i, t in enumerate(tensors):
        if t.device != dev or t.dtype not in _DTYPES or dev.type != "cuda":
            raise ValueError("clip_grad_norm: tensor %d must be float32, bfloat16 or float16 on the GPU of tensor 0 (%s), got %s on %s"
                             % (i, dev, t.dtype, t.device))
        if t.layout != torch.strided or not _dense(t):
            raise ValueError("clip_grad_norm: tensor %d is sparse or has gaps or repeated elements" % i)
        src[i], cnt[i], typ[i] = t.data_ptr(), t.numel(), _DTYPES[t.dtype]
    dst = None
    if outs is not None:
        if outs is tensors:
            dst = src
        else:
            dst = (C.c_void_p * n)()
            for i, (t, o) in enumerate(zip(tensors, outs)):
                if o.dtype != t.dtype or o.device != dev or o.shape != t.shape or (o.stride() != t.stride() and not (t.is_contiguous() and o.is_contiguous())):
                    raise ValueError("clip_grad_norm: out %d must have the shape, strides, type and device of its tensor" % i)
                dst[i] = o.data_ptr()
        spans = sorted((p, p + c * t.element_size()) for p, c, t in zip(dst, cnt, tensors) if c)
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("clip_grad_norm: a tensor is given twice, or two share memory")
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = _space(_lib.CLIP_WORKSPACE_BYTES, dev)
    _check(_lib.load().mpe_clip_grad_norm(dev.index, n, src, dst, cnt, typ, max_norm, norm.data_ptr(), ws.data_ptr(), _lib.CLIP_WORKSPACE_BYTES, _stream(dev)))
    if outs is not None:
        torch.autograd.graph.increment_version(outs)
    return norm


def _max_norm(v):
    v = float(v)
    if not v >= 0:
        raise ValueError("clip_grad_norm: max_norm must not be negative, got %r" % v)
    return v


def _tensors(tensors):
    tensors = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not tensors:
        raise ValueError("clip_grad_norm: no tensors")
    return [t.detach() for t in tensors]


def grad_norm(tensors):
    """``sqrt`` of the sum of all squares over ``tensors`` (float32, bfloat16, float16, mixed; summed in float64): a float32
    scalar on their GPU.  A tensor given twice counts twice."""
    return _clip(_tensors(tensors), 0.0, None)


def clip_grad_norm(tensors, max_norm, out):
    """Writes ``t * f`` into the tensors of ``out``, one for each of ``tensors``, ``f = max_norm / norm`` where the global norm
    is above ``max_norm`` and 1 otherwise (NaN if the norm is; an infinite norm makes it 0).  Returns the norm before
    clipping, a float32 scalar on the GPU; nothing waits for it."""
    tensors, outs = _tensors(tensors), _tensors(out)
    if len(outs) != len(tensors):
        raise ValueError("clip_grad_norm: %d tensors but %d in out" % (len(tensors), len(outs)))
    return _clip(tensors, _max_norm(max_norm), outs)


def clip_grad_norm_(parameters, max_norm):
    """Clips the gradients of ``parameters`` in place, as :func:`clip_grad_norm` does (those without one are passed over), and
    returns their norm before clipping."""
    parameters = [parameters] if torch.is_tensor(parameters) else list(parameters)
    max_norm = _max_norm(max_norm)
    grads = [p.grad.detach() for p in parameters if p.grad is not None]
    if not grads:
        raise ValueError("clip_grad_norm_: no parameter has a gradient")
    return _clip(grads, max_norm, grads)
