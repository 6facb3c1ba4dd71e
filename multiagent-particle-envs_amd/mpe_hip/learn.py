"""Trainer-side operators: what the policy update runs on a rollout that :func:`mpe_hip.gae` gave advantages to.

* ``linear``: a layer, ``f(x W^T + b) + r`` in one launch, with its gradients;
* ``ppo_loss``: the clipped policy loss with value loss and entropy bonus, with its gradients;
* ``clip_grad_norm`` / ``clip_grad_norm_`` / ``grad_norm``: the global norm over many tensors, and clipping to it.

All take GPU tensors (float32, bfloat16 or float16; there is no CPU path), enqueue on the current stream of the tensors'
device and return without synchronising.  All may be captured into a graph; a backward pass that is captured follows
autograd's own rule that no eager graph of the same leaves is alive.  Second derivatives are not available.
"""
import ctypes as C
from array import array

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.MPE_F32, torch.bfloat16: _lib.MPE_BF16, torch.float16: _lib.MPE_F16}
ACTIVATIONS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "tanh": _lib.ACT_TANH, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
               "silu": _lib.ACT_SILU}


_ROW_MAX = 1 << 22      # the longest row stride the kernels take


def _raw_stream():
    """index of a device -> handle of its current stream; torch's own getter costs a microsecond more by making an object."""
    fn = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return fn if fn is not None else lambda index: torch.cuda.current_stream(index).cuda_stream


_stream = _raw_stream()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _check(code):
    if code != 0:
        _lib.check(None, code)


def _dtype(t, what):
    if not t.is_cuda:
        raise ValueError("%s needs GPU tensors; there is no CPU path" % what)
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError("%s takes float32, bfloat16 or float16, not %s" % (what, t.dtype))
    return code


def _rows(t, cols):
    """``(matrix, row stride)``: ``t`` as rows of ``cols`` contiguous elements (any row stride >= cols), copied only if it has to be."""
    if t.is_contiguous():
        return t, cols
    m = t if t.dim() == 2 else t.reshape(-1, cols)
    rows, (ld, inner) = m.shape[0], m.stride()
    if (cols > 1 and inner != 1) or (rows > 1 and not cols <= ld <= _ROW_MAX):
        return m.contiguous(), cols
    return m, ld if rows > 1 else cols      # a single row's stride says nothing


def _rows_or_one(t, cols):
    """As _rows, but one row of a vector's length or more that is repeated by ``expand`` stays one row (stride 0)."""
    if cols >= 8 and not t.is_contiguous() and t.dim() >= 2 and t.numel() > 0 and t.stride(-1) == 1 \
            and all(s == 0 or n == 1 for s, n in zip(t.stride()[:-1], t.shape[:-1])):
        return t, 0
    return _rows(t, cols)


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
    x2, ldx = _rows(x, k)
    w2, ldw = _rows(weight, k)
    m = x.numel() // k
    dev = x.device
    y = torch.empty(x.shape[:-1] + (n,), dtype=x.dtype, device=dev)
    pre = torch.empty(m, n, dtype=x.dtype if act == _lib.ACT_RELU else torch.float32, device=dev) if keep_pre else None
    r2, ldr = (None, 0) if residual is None else _rows_or_one(residual, n)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    ws_bytes = _workspace(code, act, m, n, k)[0]
    ws = _space(ws_bytes, dev)
    _check(_lib.load().mpe_linear_forward(dev.index, code, act, m, n, k, x2.data_ptr(), ldx, w2.data_ptr(), ldw, _ptr(bias), _ptr(r2), ldr,
                                          y.data_ptr(), n, _ptr(pre), _ptr(ws), ws_bytes, _stream(dev.index)))
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
            x2, ldx = _rows(x, k)
            w2, ldw = _rows(weight, k)
            m = x.numel() // k
            dev = x.device
            dy2, lddy = _rows_or_one(dy, n)
            dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
            dw = torch.empty(n, k, dtype=x.dtype, device=dev) if need_w else None
            db = torch.empty(n, dtype=x.dtype, device=dev) if need_b else None
            ws_bytes = _workspace(ctx.code, ctx.act, m, n, k)[1]
            ws = _space(ws_bytes, dev)
            _check(_lib.load().mpe_linear_backward(dev.index, ctx.code, ctx.act, m, n, k, dy2.data_ptr(), lddy, x2.data_ptr(), ldx, w2.data_ptr(),
                                                   ldw, _ptr(pre), _ptr(dx), k, _ptr(dw), _ptr(db), _ptr(ws), ws_bytes, _stream(dev.index)))
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
    shape, wshape = x.shape, weight.shape
    if len(shape) < 1 or len(wshape) != 2 or shape[-1] != wshape[1] or wshape[0] < 1 or wshape[1] < 1:
        raise ValueError("linear: x [..., k] and weight [n, k], n and k at least 1; got %s and %s" % (tuple(shape), tuple(wshape)))
    n, dt, dev = wshape[0], x.dtype, x.device
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError("linear: bias must have shape (%d,), got %s" % (n, tuple(bias.shape)))
    if residual is not None and residual.shape != shape[:-1] + (n,):
        raise ValueError("linear: residual must have the result's shape %s, got %s" % (tuple(shape[:-1]) + (n,), tuple(residual.shape)))
    needs = x.requires_grad or weight.requires_grad
    for t in (weight, bias, residual):
        if t is not None:
            if t.dtype != dt or t.device != dev:
                raise ValueError("linear: all tensors must share x's type and device (%s, %s)" % (dt, dev))
            needs = needs or t.requires_grad
    if needs and torch.is_grad_enabled():
        return _Linear.apply(x, weight, bias, residual, act, code)
    return _linear_forward(x, weight, bias, residual, act, code, False)[0]


# ---- ppo_loss -------------------------------------------------------------------------------------------------------------

class _PpoLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, actions, old_logp, adv, old_values, returns, mask, weights, coefs, code):
        v = logits.shape[-1]
        l2, ld = _rows(logits, v)
        dev = logits.device
        loss, stats = torch.empty((), dtype=torch.float32, device=dev), torch.empty(6, dtype=torch.float32, device=dev)
        ws = torch.empty(_lib.PPO_WORKSPACE_BYTES, dtype=torch.uint8, device=dev)
        val = values if values is None or values.is_contiguous() else values.contiguous()
        m2, ldm = (None, 0) if mask is None else _rows(mask, v)
        args = (dev.index, code, logits.numel() // v, v, l2.data_ptr(), ld, actions.data_ptr(), actions.element_size(), old_logp.data_ptr(), adv.data_ptr(),
                _ptr(m2), ldm, _ptr(weights), _ptr(val), _ptr(old_values), _ptr(returns)) + coefs
        _check(_lib.load().mpe_ppo_loss_forward(*args, loss.data_ptr(), stats.data_ptr(), ws.data_ptr(), _lib.PPO_WORKSPACE_BYTES, _stream(dev.index)))
        ctx.args = args
        ctx.save_for_backward(logits, values, stats, actions, old_logp, adv, old_values, returns, mask, weights)
        ctx.kept = (l2, val, m2)        # what args point to, where it is a copy
        ctx.mark_non_differentiable(stats)
        return loss, stats

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, _):
        logits, values, stats = ctx.saved_tensors[:3]       # raises where an input was written since
        need_l, need_v = ctx.needs_input_grad[0], ctx.needs_input_grad[1] and values is not None
        dlogits = dvalues = None
        if need_l or need_v:
            dev = logits.device
            dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
            if need_v:
                dvalues = torch.empty(values.shape, dtype=torch.float32, device=dev)
            if grad.dtype != torch.float32:
                grad = grad.to(torch.float32)
            _check(_lib.load().mpe_ppo_loss_backward(*ctx.args, stats.data_ptr(), grad.data_ptr(), dlogits.data_ptr(), logits.shape[-1], _ptr(dvalues),
                                                     _stream(dev.index)))
        return (dlogits if need_l else None, dvalues) + (None,) * 9


def _side(name, t, dtype, shape, dev):
    """A tensor that goes with the logits, checked and contiguous."""
    if t is None:
        return None
    if t.dtype != dtype:
        raise ValueError("ppo_loss: %s must be %s, not %s" % (name, str(dtype).replace("torch.", ""), t.dtype))
    if t.shape != shape or t.device != dev:
        raise ValueError("ppo_loss: %s must have shape %s on %s, got %s on %s" % (name, tuple(shape), dev, tuple(t.shape), t.device))
    return t if t.is_contiguous() else t.contiguous()


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
    shape, dev = logits.shape, logits.device
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError("ppo_loss: logits must be [..., v] with v at least 1, got %s" % (tuple(shape),))
    lead, f32 = shape[:-1], torch.float32
    if (values is None) != (old_values is None) or (values is None) != (returns is None):
        raise ValueError("ppo_loss: values, old_values and returns go together")
    if actions.dtype not in (torch.int32, torch.int64):
        raise ValueError("ppo_loss: actions must be int32 or int64, not %s" % actions.dtype)
    if weights is not None and weights.dtype == torch.bool:
        weights = weights.float()
    if action_mask is not None:
        if action_mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError("ppo_loss: action_mask must be bool or uint8, not %s" % action_mask.dtype)
        if action_mask.shape != shape or action_mask.device != dev:
            raise ValueError("ppo_loss: action_mask must have shape %s on %s, got %s on %s" % (tuple(shape), dev, tuple(action_mask.shape), action_mask.device))
    if values is not None and (values.dtype != f32 or values.shape != lead or values.device != dev):
        raise ValueError("ppo_loss: values must be float32 of shape %s on %s, got %s %s on %s" % (tuple(lead), dev, values.dtype, tuple(values.shape), values.device))
    clip, value_clip = float(clip), -1.0 if value_clip is None else float(value_clip)
    if not clip >= 0 or not (value_clip >= 0 or value_clip == -1.0):
        raise ValueError("ppo_loss: clip and value_clip must not be negative")
    loss, stats = _PpoLoss.apply(logits, values, _side("actions", actions, actions.dtype, lead, dev), _side("old_logp", old_logp, f32, lead, dev),
                                 _side("advantages", advantages, f32, lead, dev), _side("old_values", old_values, f32, lead, dev),
                                 _side("returns", returns, f32, lead, dev), action_mask, _side("weights", weights, f32, lead, dev),
                                 (clip, value_clip, float(value_coef), float(entropy_coef)), code)
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
    dev = tensors[0].device
    types = [t.dtype for t in tensors]
    for i, t in enumerate(tensors):
        if t.device != dev or not t.is_cuda or types[i] not in _DTYPES:
            raise ValueError("clip_grad_norm: tensor %d must be float32, bfloat16 or float16 on the GPU of tensor 0 (%s), got %s on %s"
                             % (i, dev, types[i], t.device))
        if t.layout != torch.strided or not (t.is_contiguous() or _dense(t)):
            raise ValueError("clip_grad_norm: tensor %d is sparse or has gaps or repeated elements" % i)
    src = array("Q", [t.data_ptr() for t in tensors])
    counts = array("q", [t.numel() for t in tensors])
    codes = array("i", [_DTYPES[d] for d in types])
    dst = None
    if outs is tensors:
        dst = src
    elif outs is not None:
        for i, (t, o) in enumerate(zip(tensors, outs)):
            if o.dtype != types[i] or o.device != dev or o.shape != t.shape or not (o.is_contiguous() and t.is_contiguous() or o.stride() == t.stride()):
                raise ValueError("clip_grad_norm: out %d must have the shape, strides, type and device of its tensor" % i)
        dst = array("Q", [o.data_ptr() for o in outs])
    if dst is not None:
        end = 0
        for p, bytes_ in sorted([(p, c * (4 if d == 0 else 2)) for p, c, d in zip(dst, counts, codes) if c]):
            if p < end:
                raise ValueError("clip_grad_norm: a tensor is given twice, or two share memory")
            end = p + bytes_
    norm = torch.empty((), dtype=torch.float32, device=dev)
    ws = torch.empty(_lib.CLIP_WORKSPACE_BYTES, dtype=torch.uint8, device=dev)
    _check(_lib.load().mpe_clip_grad_norm(dev.index, len(tensors), src.buffer_info()[0], dst.buffer_info()[0] if dst is not None else None,
                                          counts.buffer_info()[0], codes.buffer_info()[0], max_norm, norm.data_ptr(), ws.data_ptr(),
                                          _lib.CLIP_WORKSPACE_BYTES, _stream(dev.index)))
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
    return tensors


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
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        raise ValueError("clip_grad_norm_: no parameter has a gradient")
    return _clip(grads, max_norm, grads)
