"""The linear layer with what surrounds it as one operator: bias, activation and residual, any sizes, with gradients.

The Linear layers of the trunk, the encoders and the heads are fused at their own widths (and the latter two forward-only); this is one on its
own, for heads and layers of other shapes that are trained.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _capi
from . import _ops, _update_ops
from ._sequence_ops import activation_code


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: Optional[str] = None,
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual, on the tensor cores, differentiable in all four.

    Args:
        x: (.., K) float32, bfloat16 or float16.
        weight: (N, K) as ``nn.Linear`` stores it, bias: (N): x's type or float32.  A call of 16-bit x rounds float32 weights to x's
            type as autocast does (gradients are float32 then), a float32 bias is added as it is.
        activation: None, "silu" or "gelu" (erf).
        residual: (.., N) of x's type.

    Returns:
        (.., N) in x's type, rounded once.  16-bit calls: products of 16-bit operands summed in float32; the gradient before the activation is
        rounded to x's type as an operand of the next products, but not for the bias's gradient, its sum.  Between forward and backward, bfloat16
        calls keep the activation's slopes in 16 bits (relative 2^-12), calls with a float32 bias, float16 and float32 ones the sums in 32.  float32 calls: float32
        products, of numbers in pieces, so that an infinity, or a number above 3.39e38, comes out as NaN.
    """
    act = activation_code("linear", activation, (None, "silu", "gelu"))
    if _ops.direct(x):
        return _capi.host.linear(x, weight, bias, residual, act)
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual))
    return _update_ops.linear(x, weight, bias, residual, act, keep)[0]
