"""Trainer-side operators: what the policy update runs on a rollout that :func:`mpe_hip.gae` gave advantages to.

* ``linear``: a layer, ``f(x W^T + b) + r`` in one launch, with its gradients;
* ``ppo_loss``: the clipped policy loss with value loss and entropy bonus, with its gradients;
* ``clip_grad_norm`` / ``clip_grad_norm_`` / ``grad_norm``: the global norm over many tensors, and clipping to it.

All take GPU tensors (float32, bfloat16 or float16; there is no CPU path), enqueue on the current stream of the tensors'
device and return without synchronising.  All may be captured into a graph; a backward pass that is captured follows
autograd's own rule that no eager graph of the same leaves is alive.  Second derivatives and forward-mode derivatives are not
available: both are refused.

The calls and their autograd nodes are C++ (csrc/mpe_torch.cpp, built into ``_native.so`` next to the library): an operator
of a few microseconds would otherwise wait for the interpreter.
"""
import ctypes as C

import torch

from . import _lib

ACTIVATIONS = {None: _lib.ACT_NONE, "none": _lib.ACT_NONE, "tanh": _lib.ACT_TANH, "relu": _lib.ACT_RELU, "gelu": _lib.ACT_GELU,
               "silu": _lib.ACT_SILU}

_module = None


def _native():
    """The compiled module, bound to the library that _lib has loaded."""
    global _module
    if _module is None:
        lib = _lib.load()
        try:
            from . import _native as module
        except ImportError as e:
            raise ImportError("mpe_hip/_native.so is missing or does not load (%s): run `python __graft_entry__.py build` at the repository "
                              "root; there is no fallback." % e) from e
        names = ("mpe_last_error", "mpe_linear_workspace", "mpe_linear_forward", "mpe_linear_backward", "mpe_ppo_loss_forward",
                 "mpe_ppo_loss_backward", "mpe_clip_grad_norm")
        module.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in names}, _lib.MpeError)
        _module = module
    return _module


def linear(x, weight, bias=None, activation=None, residual=None):
    """``activation(x @ weight.T + bias) + residual`` in one launch, differentiable in all four.

    ``x`` ``[..., k]`` (rows may be strided: ``env.obs_n[i]`` is taken as it lies), ``weight`` ``[n, k]``, ``bias`` ``[n]``,
    ``residual`` of the result's shape ``[..., n]`` (an expanded tensor will do); all of one type (float32, bfloat16,
    float16) on one GPU.  ``activation``: None / "none", "tanh", "relu", "gelu" (by erf) or "silu".  Sums are in float32 or
    better, with one rounding to the type at the end; float32 products are as exact as float32 multiplications, of numbers
    above 2^-109.  For the backward pass float32 and float16 keep float32 pre-activations, bfloat16 keeps the slopes in float16
    (nothing is kept for none, and for relu and float32 tanh without residual); 16-bit gradients are sums of dz with twice the
    type's bits, rounded once."""
    try:
        act = ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError("linear: activation must be one of none, tanh, relu, gelu, silu; got %r" % (activation,)) from None
    return (_module or _native()).linear(x, weight, bias, residual, act)


def ppo_loss(logits, actions, old_logp, advantages, values=None, old_values=None, returns=None, action_mask=None, weights=None, clip=0.2,
             value_clip=None, value_coef=0.5, entropy_coef=0.01):
    """The clipped policy loss of a rollout, differentiable in ``logits`` and ``values``.

    ``logits`` ``[..., v]`` (float32, bfloat16, float16; rows may be strided); everything else has its leading shape:
    ``actions`` int32 / int64, ``old_logp`` and ``advantages`` float32, optionally ``values``, ``old_values`` and
    ``returns`` float32 (together), ``action_mask`` bool / uint8 ``[..., v]`` (0 forbids a move) and ``weights`` float32
    (none negative) / bool.  Per decision, with the softmax over the allowed moves: ``q = exp(logp - old_logp)``,
    ``s = min(q A, clamp(q, 1 - clip, 1 + clip) A)``, the entropy ``H`` and the value loss
    ``u = max((V - R)^2, (V0 + clamp(V - V0, -value_clip, value_clip) - R)^2) / 2`` (``value_clip`` None: ``(V - R)^2 / 2``);
    ``loss = sum w (-s + value_coef u - entropy_coef H) / sum w``.

    A decision is left out, with zero gradients, if its weight is 0 or its action lies outside ``[0, v)``, is forbidden or
    has the logit -infinity (so also where no move is left).  Returns ``(loss, stats)``: a float32 scalar and the float32 means
    ``[-s, u, H, (logp - old_logp)^2 / 2, share of clipped decisions]``."""
    return (_module or _native()).ppo_loss(logits, actions, old_logp, advantages, values, old_values, returns, action_mask, weights, clip,
                                           value_clip, value_coef, entropy_coef)


def _list(tensors):
    return [tensors] if torch.is_tensor(tensors) else list(tensors)


def grad_norm(tensors):
    """``sqrt`` of the sum of all squares over ``tensors`` (float32, bfloat16, float16, mixed; summed in float64): a float32
    scalar on their GPU, which carries no gradient.  A tensor given twice counts twice."""
    return (_module or _native()).clip(_list(tensors), 0.0, None)


def clip_grad_norm(tensors, max_norm, out):
    """Writes ``t * f`` into the tensors of ``out``, one for each of ``tensors``, ``f = max_norm / norm`` where the global norm
    is above ``max_norm`` and 1 otherwise (NaN if the norm is; an infinite norm makes it 0).  Returns the norm before
    clipping, a float32 scalar on the GPU; nothing waits for it.  A tensor may be its own ``out``; any other overlap of an
    ``out`` with a tensor is refused.  Nothing here is differentiable: an ``out`` that requires gradients is refused
    unless they are off."""
    return (_module or _native()).clip(_list(tensors), max_norm, _list(out))


def clip_grad_norm_(parameters, max_norm):
    """Clips the gradients of ``parameters`` in place, as :func:`clip_grad_norm` does (those without one are passed over), and
    returns their norm before clipping."""
    grads = [p.grad for p in _list(parameters) if p.grad is not None]
    if not grads:
        raise ValueError("clip_grad_norm_: no parameter has a gradient")
    return (_module or _native()).clip(grads, max_norm, grads)
