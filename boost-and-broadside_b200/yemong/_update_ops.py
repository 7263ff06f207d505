"""Opaque ``torch.library`` operators of an update's end (``policy_loss.py``), for callers that have to see them: a compiler, a
tracer, a dispatch mode.  Same reason and same form as ``_ops.py``; eager calls go to the native code (csrc/host_update.cpp)
directly, autograd nodes included.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from .. import _capi


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
            logits.new_empty(4 + rows * (2 * max(1, len(sizes)) + 1), **f))


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
