"""The gated feed-forward block as an operator: any width and hidden size, with gradients.

``GatedMLP`` (attention.py:21-37 of the reference) inside the trunk is fused into the sublayers at their width; this is the block
on its own, for layers outside the trunk and for ``GatedMLP`` where it is differentiated.
"""

from __future__ import annotations

import torch

from .. import _capi
from . import _ops, _sequence_ops
from ._sequence_ops import activation_code


def gated_mlp(x: torch.Tensor, gate_w: torch.Tensor, up_w: torch.Tensor, down_w: torch.Tensor, *, activation: str = "gelu") -> torch.Tensor:
    """down_w (act(gate_w x) * (up_w x)), on the tensor cores, differentiable in all four.

    Args:
        x: (.., D) float32, bfloat16 or float16.
        gate_w, up_w: (F, D); down_w: (D, F), as ``nn.Linear`` stores them: x's type, or float32, which a
            call of 16-bit x rounds to x's type as autocast does (gradients are float32 then).
        activation: "gelu" (erf) or "silu".

    Returns:
        (.., D) in x's type.  16-bit calls: products of 16-bit operands summed in float32, the hidden activations and their
        gradients rounded to x's type as operands of the next product.  float32 calls: float32 products, of numbers in pieces, so that
        an infinity, or a number above 3.39e38, comes out as NaN.
    """
    act = activation_code("gated_mlp", activation, ("gelu", "silu"))
    if _ops.direct(x):
        return _capi.host.gated_mlp(x, gate_w, up_w, down_w, act)
    keep = torch.is_grad_enabled() and any(t.requires_grad for t in (x, gate_w, up_w, down_w))
    return _sequence_ops.gated_mlp(x, gate_w, up_w, down_w, act, keep)[0]
