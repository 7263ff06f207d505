"""The clipped policy loss with a KL term, of a head's logits, with their gradient.

Beside ``evaluate_action`` (policy.py:578-602 of the reference), which is forward-only and has the policy's own three slices: the policy's part of
the update's loss (ppo.py:1351) in one operator, for any number of slices and actions.
"""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

import torch

from .. import _capi
from . import _ops, _update_ops


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, old_logprob: torch.Tensor, advantages: torch.Tensor, *,
                weights: Optional[torch.Tensor] = None, ref_logprob: Optional[torch.Tensor] = None, sizes: Optional[Sequence[int]] = None,
                clip: Union[float, Tuple[float, float]] = 0.2, kl_coef: float = 0.0,
                entropy_coef: float = 0.0, grad_in_forward: bool = True) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The mean over rows of  -min(ratio A, clip(ratio) A) + kl_coef k - entropy_coef H,  differentiable in the logits.

    ``ratio`` is exp(l - old_logprob) of the log-probability l of a row's actions, k = exp(ref_logprob - l) - (ref_logprob - l) - 1 estimates the
    KL divergence from the reference policy, H is the entropy.

    Args:
        logits: (.., V) float32, bfloat16 or float16.  -inf or the type's lowest value forbids an action.
        actions: (..) int64 or int32; with ``sizes`` (.., S).  One outside of its slice makes the row's results, and the loss, NaN.
        old_logprob, advantages, ref_logprob: (..); no gradients are taken for them.
        weights: (..) bool, or floating-point weights of the mean.  Rows of weight 0 are not looked at, whatever stands in them: their
            log-probability and gradient are 0.  The loss is 0 where no row has weight.
        sizes: up to 16 distributions side by side, V in total, such as (3, 7, 2); their log-probabilities and entropies add up.
        clip: how far the ratio may go from 1, in both directions or (down, up).
        grad_in_forward: write the gradient with the forward, in one pass over the logits, where slices are wider than 64 and not float16.
            It is what the backward returns when the loss arrives there multiplied by 1; by anything else, it is computed once more.  False leaves it to
            the backward: for losses that are scaled.

    Returns:
        (loss, logprob, stats): loss () and l (..) in float32, and the means of (surrogate, k, H, whether the ratio is outside
        of its clipping), float32.  Only the loss is differentiable, once.
    """
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (low >= 0 and high >= 0):
        raise ValueError(f"policy_loss: clip must not be negative, got {clip!r}")
    if torch.is_grad_enabled():
        for name, t in (("old_logprob", old_logprob), ("advantages", advantages), ("ref_logprob", ref_logprob), ("weights", weights)):
            if t is not None and t.requires_grad:
                raise NotImplementedError(f"policy_loss is differentiable in the logits only; detach {name}")
    numbers = ([] if sizes is None else list(sizes), float(low), float(high), float(kl_coef), float(entropy_coef))
    if sizes is not None and not numbers[0]:
        raise ValueError("policy_loss: sizes must name at least one slice")
    if _ops.direct(logits):
        return _capi.host.policy_loss(logits, actions, old_logprob, advantages, ref_logprob, weights, *numbers, grad_in_forward)
    return _update_ops.policy_loss(logits, actions, old_logprob, advantages, ref_logprob, weights, *numbers)[:3]
