"""Opaque ``torch.library`` operators of the layers outside the trunk (``selective.py``, ``gated.py``), for callers
that have to see them: a compiler, a tracer, a dispatch mode.  Same reason and same form as ``_ops.py``;
eager calls go to the native code (csrc/host_operators.cpp) directly, autograd nodes included.
"""

from __future__ import annotations

from typing import List, Optional, Tuple

import torch
from torch import Tensor

from .. import _capi


_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}


def activation_code(fn: str, name: Optional[str], allowed: tuple) -> int:
    if name not in allowed:
        raise ValueError(f"{fn}: activation must be one of {allowed}, got {name!r}")
    return _ACTIVATIONS[name]


def _rows_like(x: Tensor) -> Tensor:
    """As the native code lays out a result of x's shape: step by step, or row by row where x is."""
    if x.dim() < 3 or x.stride(0) >= x.stride(1):
        return x.new_empty(x.shape)
    return x.new_empty_strided(x.shape, (x.shape[2], x.shape[0] * x.shape[2], 1))


def _given(grads: List[Tensor], has: List[bool]) -> list:
    """Gradients of a call's inputs: None for the inputs that were not given."""
    return [g if h else None for g, h in zip(grads, has)]


# ----------------------------------------------------------------------------- causal convolution


@torch.library.custom_op("bnb_b200::causal_conv", mutates_args=(), device_types="cuda")
def causal_conv(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Optional[Tensor], done: Optional[Tensor],
                lengths: Optional[Tensor], activation: int) -> Tuple[Tensor, Tensor]:
    """``bnb_causal_conv_fwd``: x (T, R, C), weight (C, K) -> (y like x, state (R, K-1, C))."""
    return _capi.host.causal_conv_forward(x, weight, bias, state, done, lengths, activation)


@causal_conv.register_fake
def _(x, weight, bias, state, done, lengths, activation):
    return _rows_like(x), weight.new_empty((x.shape[1], weight.shape[1] - 1, x.shape[2]))


@torch.library.custom_op("bnb_b200::causal_conv_backward", mutates_args=(), device_types="cuda")
def causal_conv_backward(x: Tensor, weight: Tensor, bias: Optional[Tensor], state: Optional[Tensor], done: Optional[Tensor],
                         lengths: Optional[Tensor], activation: int, dy: Optional[Tensor], dstate: Optional[Tensor]) -> List[Tensor]:
    """Gradients of x, weight, bias and state; an empty tensor for one that was not given."""
    out = _capi.host.causal_conv_backward(x, weight, bias, state, done, lengths, activation, dy, dstate)
    return [weight.new_empty(0) if g is None else g for g in out]


@causal_conv_backward.register_fake
def _(x, weight, bias, state, done, lengths, activation, dy, dstate):
    return [_rows_like(x), weight.new_empty(weight.shape), weight.new_empty(0 if bias is None else bias.shape),
            weight.new_empty(0 if state is None else state.shape)]


def _conv_context(ctx, inputs, output):
    x, weight, bias, state, done, lengths, activation = inputs
    ctx.activation = activation
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, weight, bias, state, done, lengths)


def _conv_formula(ctx, dy, dstate):
    x, weight, bias, state, done, lengths = ctx.saved_tensors
    out = causal_conv_backward(x, weight, bias, state, done, lengths, ctx.activation, dy, dstate)
    return (*_given(out, [True, True, bias is not None, state is not None]), None, None, None)


causal_conv.register_autograd(_conv_formula, setup_context=_conv_context)


@torch.library.custom_op("bnb_b200::causal_conv_step", mutates_args=("state",), device_types="cuda")
def causal_conv_step(x: Tensor, state: Tensor, weight: Tensor, bias: Optional[Tensor], reset: Optional[Tensor], activation: int) -> Tensor:
    """One token a row: x (R, C) -> y (R, C); state (R, K-1, C) moves on in place."""
    return _capi.host.causal_conv_step(x, state, weight, bias, reset, activation)


@causal_conv_step.register_fake
def _(x, state, weight, bias, reset, activation):
    return x.new_empty(x.shape)


# ----------------------------------------------------------------------------- selective scan


@torch.library.custom_op("bnb_b200::selective_scan", mutates_args=(), device_types="cuda")
def selective_scan(u: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor],
                   delta_bias: Optional[Tensor], state: Optional[Tensor], done: Optional[Tensor], lengths: Optional[Tensor],
                   softplus: bool, keep: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """``bnb_selective_scan_fwd``: u, delta, z (T, R, C), A (C, N), B, C (T, R, G, N) -> (y like u, state (R, C, N), the
    states kept for the backward: empty without ``keep``)."""
    return _capi.host.selective_scan_forward(u, delta, A, B, C, D, z, delta_bias, state, done, lengths, softplus, keep)


def _kept_numel(T: int, R: int, C: int, N: int) -> int:
    lanes = 4
    while lanes < N:
        lanes *= 2
    return (T + 7) // 8 * R * C * lanes


@selective_scan.register_fake
def _(u, delta, A, B, C, D, z, delta_bias, state, done, lengths, softplus, keep):
    (T, R, W), N = u.shape, A.shape[1]
    return _rows_like(u), A.new_empty((R, W, N)), A.new_empty(_kept_numel(T, R, W, N) if keep else 0)


@torch.library.custom_op("bnb_b200::selective_scan_backward", mutates_args=(), device_types="cuda")
def selective_scan_backward(u: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], z: Optional[Tensor],
                            delta_bias: Optional[Tensor], state: Optional[Tensor], done: Optional[Tensor], lengths: Optional[Tensor],
                            softplus: bool, kept: Tensor, dy: Optional[Tensor], dstate: Optional[Tensor]) -> List[Tensor]:
    """Gradients of u, delta, A, B, C, D, z, delta_bias and state; an empty tensor for one that was not given."""
    out = _capi.host.selective_scan_backward(u, delta, A, B, C, D, z, delta_bias, state, done, lengths, softplus, kept, dy, dstate)
    return [A.new_empty(0) if g is None else g for g in out]


@selective_scan_backward.register_fake
def _(u, delta, A, B, C, D, z, delta_bias, state, done, lengths, softplus, kept, dy, dstate):
    like = lambda t: A.new_empty(0) if t is None else A.new_empty(t.shape)  # noqa: E731
    return [_rows_like(u), _rows_like(delta), like(A), B.new_empty(B.shape), C.new_empty(C.shape), like(D),
            A.new_empty(0) if z is None else _rows_like(z), like(delta_bias), like(state)]


def _scan_context(ctx, inputs, output):
    *tensors, softplus, keep = inputs
    ctx.softplus, ctx.keep = softplus, keep
    ctx.mark_non_differentiable(output[2])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(*tensors, output[2])


def _scan_formula(ctx, dy, dstate, _dkept):
    *tensors, kept = ctx.saved_tensors
    if not ctx.keep:
        raise RuntimeError("selective_scan was called without keeping the states that its backward reads")
    out = selective_scan_backward(*tensors, ctx.softplus, kept, dy, dstate)
    return (*_given(out, [t is not None for t in tensors[:9]]), None, None, None, None)


selective_scan.register_autograd(_scan_formula, setup_context=_scan_context)


@torch.library.custom_op("bnb_b200::selective_step", mutates_args=("state",), device_types="cuda")
def selective_step(u: Tensor, delta: Tensor, A: Tensor, B: Tensor, C: Tensor, D: Optional[Tensor], state: Tensor, z: Optional[Tensor],
                   delta_bias: Optional[Tensor], reset: Optional[Tensor], softplus: bool) -> Tensor:
    """One token a row: u (R, C) -> y (R, C); state (R, C, N) moves on in place."""
    return _capi.host.selective_step(u, delta, A, B, C, D, state, z, delta_bias, reset, softplus)


@selective_step.register_fake
def _(u, delta, A, B, C, D, state, z, delta_bias, reset, softplus):
    return u.new_empty(u.shape)


# ----------------------------------------------------------------------------- gated feed-forward block


@torch.library.custom_op("bnb_b200::gated_mlp", mutates_args=(), device_types="cuda")
def gated_mlp(x: Tensor, gate_w: Tensor, up_w: Tensor, down_w: Tensor, activation: int, keep: bool) -> Tuple[Tensor, Tensor]:
    """``bnb_gated_block_fwd``: x (.., D) -> (y like x, what the backward reads: empty without ``keep``)."""
    return _capi.host.gated_mlp_forward(x, gate_w, up_w, down_w, activation, keep)


@gated_mlp.register_fake
def _(x, gate_w, up_w, down_w, activation, keep):
    # as bnb_gated_block_kept_bytes: narrow 16-bit calls compute g and u once more and keep nothing
    recomputes = x.dtype != torch.float32 and x.shape[-1] <= 512
    rows = x.numel() // x.shape[-1]
    kept = 8 * ((rows + 31) // 32 * 32) * ((gate_w.shape[0] + 31) // 32 * 32)
    return x.new_empty(x.shape), x.new_empty(kept if keep and not recomputes else 0, dtype=torch.uint8)


@torch.library.custom_op("bnb_b200::gated_mlp_backward", mutates_args=(), device_types="cuda")
def gated_mlp_backward(x: Tensor, gate_w: Tensor, up_w: Tensor, down_w: Tensor, activation: int, kept: Tensor, dy: Tensor) -> List[Tensor]:
    """Gradients of x, gate_w, up_w and down_w."""
    return _capi.host.gated_mlp_backward(x, gate_w, up_w, down_w, activation, kept, dy)


@gated_mlp_backward.register_fake
def _(x, gate_w, up_w, down_w, activation, kept, dy):
    return [t.new_empty(t.shape) for t in (x, gate_w, up_w, down_w)]


def _gated_context(ctx, inputs, output):
    x, gate_w, up_w, down_w, activation, keep = inputs
    ctx.activation, ctx.keep = activation, keep
    ctx.mark_non_differentiable(output[1])
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(x, gate_w, up_w, down_w, output[1])


def _gated_formula(ctx, dy, _dkept):
    if not ctx.keep:
        raise RuntimeError("gated_mlp was called without keeping what its backward reads")
    x, gate_w, up_w, down_w, kept = ctx.saved_tensors
    if dy is None:
        return (None,) * 6
    return (*gated_mlp_backward(x, gate_w, up_w, down_w, ctx.activation, kept, dy), None, None)


gated_mlp.register_autograd(_gated_formula, setup_context=_gated_context)
