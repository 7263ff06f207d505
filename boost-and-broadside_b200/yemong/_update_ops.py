"""Opaque ``torch.library`` operators of an update's end (``linear.py``, ``policy_loss.py``), for callers that have to see them: a compiler, a
tracer, a dispatch mode.  Same reason and same form as ``_ops.py``; eager calls go to the native code (csrc/host_update.cpp)
directly, autograd nodes included.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from .. import _capi


# ----------------------------------------------------------------------------- linear layer


@torch.library.custom_op("bnb_b200::linear", mutates_args=(), device_types="cuda")
def linear(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], activation: int, keep: bool) -> Tuple[Tensor, Tensor]:
    """``bnb_linear_fwd``: x (.., K), weight (N, K) -> (y (.., N), what the backward reads: empty without ``keep``)."""
    return _capi.host.linear_forward(x, weight, bias, residual, activation, keep)


@linear.register_fake
def _(x, weight, bias, residual, activation, keep):
    # as bnb_linear_kept_bytes: slopes in 16 bits, or z in 32; without an activation nothing
    rows = x.numel() // x.shape[-1]
    kept = (2 if x.dtype == torch.bfloat16 and (bias is None or bias.dtype == x.dtype) else 4) * ((rows + 31) // 32 * 32) * ((weight.shape[0] + 31) // 32 * 32)
    return x.new_empty((*x.shape[:-1], weight.shape[0])), x.new_empty(kept if keep and activation else 0, dtype=torch.uint8)


@torch.library.custom_op("bnb_b200::linear_backward", mutates_args=(), device_types="cuda")
def linear_backward(x: Tensor, weight: Tensor, bias: Optional[Tensor], activation: int, kept: Tensor, dy: Tensor, want_x: bool, want_weight: bool,
                    want_bias: bool) -> List[Tensor]:
    """Gradients of x, weight and bias; an empty tensor for one that is not wanted or was not given."""
    out = _capi.host.linear_backward(x, weight, bias, activation, kept, dy, want_x, want_weight, want_bias)
    return [x.new_empty(0) if g is None else g for g in out]


@linear_backward.register_fake
def _(x, weight, bias, activation, kept, dy, want_x, want_weight, want_bias):
    like = lambda t, wanted: x.new_empty(0) if t is None or not wanted else t.new_empty(t.shape)  # noqa: E731
    return [like(x, want_x), like(weight, want_weight), like(bias, want_bias)]


def _linear_context(ctx, inputs, output):
    x, weight, bias, residual, activation, keep = inputs
    ctx.activation, ctx.keep, ctx.has_residual = activation, keep, residual is not None
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, bias, output[1])


def _linear_formula(ctx, dy, _dkept):
    if not ctx.keep:
        raise RuntimeError("linear was called without keeping what its backward reads")
    x, weight, bias, kept = ctx.saved_tensors
    if dy is None:
        return (None,) * 6
    want = ctx.needs_input_grad
    wants = (want[0], want[1], want[2] and bias is not None)
    grads = linear_backward(x, weight, bias, ctx.activation, kept, dy, *wants)
    return (*(g if w else None for g, w in zip(grads, wants)), dy if ctx.has_residual else None, None, None)


linear.register_autograd(_linear_formula, setup_context=_linear_context)


# ----------------------------------------------------------------------------- policy loss


@torch.library.custom_op("bnb_b200::policy_loss", mutates_args=(), device_types="cuda")
def policy_loss(logits: Tensor, actions: Tensor, old_logprob: Tensor, advantages: Tensor, ref_logprob: Optional[Tensor], weights: Optional[Tensor],
                sizes: List[int], clip_low: float, clip_high: float, kl_coef: float, entropy_coef: float) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """``bnb_policy_loss_fwd``: logits (.., V) -> (loss (), log-probabilities (..), means (4), what the backward reads)."""
    return _capi.host.policy_loss_forward(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef,
                                          entropy_coef)


@policy_loss.register_fake
def _(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef):
    rows = logits.numel() // logits.shape[-1]
    f = {"dtype": torch.float32}
    return (logits.new_empty((), **f), logits.new_empty(logits.shape[:-1], **f), logits.new_empty(4, **f),
            logits.new_empty(4 + rows * (2 * max(1, len(sizes)) + 2), **f))


@torch.library.custom_op("bnb_b200::policy_loss_backward", mutates_args=(), device_types="cuda")
def policy_loss_backward(logits: Tensor, actions: Tensor, old_logprob: Tensor, advantages: Tensor, ref_logprob: Optional[Tensor],
                         weights: Optional[Tensor], sizes: List[int], clip_low: float, clip_high: float, kl_coef: float, entropy_coef: float,
                         kept: Tensor, dloss: Tensor) -> Tensor:
    """The gradient of the logits."""
    return _capi.host.policy_loss_backward(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef,
                                           entropy_coef, kept, dloss)


@policy_loss_backward.register_fake
def _(logits, actions, old_logprob, advantages, ref_logprob, weights, sizes, clip_low, clip_high, kl_coef, entropy_coef, kept, dloss):
    return logits.new_empty(logits.shape)


def _policy_context(ctx, inputs, output):
    *tensors, sizes, clip_low, clip_high, kl_coef, entropy_coef = inputs
    ctx.numbers = (sizes, clip_low, clip_high, kl_coef, entropy_coef)
    ctx.mark_non_differentiable(*output[1:])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*tensors, output[3])


def _policy_formula(ctx, dloss, *_others):
    *tensors, kept = ctx.saved_tensors
    d = None if dloss is None else policy_loss_backward(*tensors, *ctx.numbers, kept, dloss)
    return (d,) + (None,) * 10


policy_loss.register_autograd(_policy_formula, setup_context=_policy_context)
