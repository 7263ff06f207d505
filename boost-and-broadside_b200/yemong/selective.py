"""Recurrent operators for layers outside the trunk: the short causal convolution and the selective state
space recurrence, for whole sequences (with gradients) and for single tokens (state in place).

They take the place of conv + RG-LRU of the Griffin sublayer (griffin.py:249-286) where a layer
wants a larger state whose decay depends on the input, and follow that sublayer's conventions: time-major sequences
(T, R, C) whose rows are sequences of their own, float32 states that the caller carries, ``done`` marking
the step an episode ends at (nothing before it reaches a later step; an end at the last step leaves the returned
state alone, as in ``YemongTrunk.sequence``, and the caller clears it before the next call: ``reset`` of the
single-token forms does).

Activations may be float32, bfloat16 or float16 and strided (columns of a projection's output, batch-major
tensors transposed), innermost stride 1; parameters and states are float32.  All arithmetic is float32, rounded
once on the way out.
"""

from __future__ import annotations

import torch

from .. import _capi
from . import _ops, _sequence_ops

_ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2}


def activation_code(fn: str, name: str | None, allowed: tuple) -> int:
    if name not in allowed:
        raise ValueError(f"{fn}: activation must be one of {allowed}, got {name!r}")
    return _ACTIVATIONS[name]


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, state: torch.Tensor | None = None,
                done: torch.Tensor | None = None, lengths: torch.Tensor | None = None,
                activation: str | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Causal depthwise convolution over time: y[t] = act(bias + sum_j weight[:, K-1-j] x[t-j]).

    Args:
        x: (T, R, C).
        weight: (C, K) float32, 2 <= K <= 4, the newest tap last (``nn.Conv1d.weight[:, 0]``).
        bias: (C,) float32.
        state: (R, K-1, C) float32, the inputs before step 0, oldest first; zeros if not given.
        done: (T, R) bool, an episode ends behind the step: its inputs are no taps of later steps.
        lengths: (R,) int, the steps of each row: what stands behind them is not read, y is zero there,
            and the returned state is that of the row's last step.  Clamped to 0..T.
        activation: None or "silu".

    Returns:
        y (T, R, C) in x's type and the state (R, K-1, C) behind the last step.
    """
    act = activation_code("causal_conv", activation, (None, "silu"))
    if _ops.direct(x):
        return _capi.host.causal_conv(x, weight, bias, state, done, lengths, act)
    return _sequence_ops.causal_conv(x, weight, bias, state, done, lengths, act)


def _forward_only(fn: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"{fn} updates its state in place and is forward-only; call it under torch.no_grad()")


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *,
                     reset: torch.Tensor | None = None, activation: str | None = None) -> torch.Tensor:
    """``causal_conv`` for one token a row: x (R, C) -> y (R, C).  ``state`` (R, K-1, C) float32, contiguous, moves
    on in place; rows of ``reset`` (R,) bool start from zeros.  Forward only."""
    act = activation_code("causal_conv_step", activation, (None, "silu"))
    _forward_only("causal_conv_step", x, state, weight, bias)
    run = _capi.host if _ops.direct(x) else _sequence_ops
    return run.causal_conv_step(x, state, weight, bias, reset, act)


def _grouped(fn: str, name: str, t: torch.Tensor, dims: int) -> torch.Tensor:
    """B or C with its group dimension: one group if it has none."""
    if t.dim() == dims:
        return t.unsqueeze(-2)
    if t.dim() != dims + 1:
        raise RuntimeError(f"{fn}: {name} must have {dims} dims, or {dims + 1} with groups, got {tuple(t.shape)}")
    return t


def selective_scan(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: torch.Tensor | None = None, *,
                   z: torch.Tensor | None = None, delta_bias: torch.Tensor | None = None, softplus: bool = False,
                   state: torch.Tensor | None = None, done: torch.Tensor | None = None,
                   lengths: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The selective state space recurrence.  Per row, channel and state n of N:

        p = delta + delta_bias, through softplus if asked for
        h_n = exp(p A_n) h_n + p u B_n
        y = (sum_n C_n h_n + D u) silu(z)            (the gate only if z is given)

    Args:
        u, delta, z: (T, R, C) of one type.
        A: (C, N) float32, 1 <= N <= 64; negative where the state is to decay.
        B, C: (T, R, N), or (T, R, G, N) with G groups of channels that share them, in u's type.
        D, delta_bias: (C,) float32.
        state: (R, C, N) float32, h before step 0; zeros if not given.
        done, lengths: as for ``causal_conv``.

    Returns:
        y (T, R, C) in u's type and the state (R, C, N) behind the last step.
    """
    B, C = _grouped("selective_scan", "B", B, 3), _grouped("selective_scan", "C", C, 3)
    if _ops.direct(u):
        return _capi.host.selective_scan(u, delta, A, B, C, D, z, delta_bias, state, done, lengths, softplus)
    inputs = (u, delta, A, B, C, D, z, delta_bias, state)
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs)
    y, new_state, _ = _sequence_ops.selective_scan(*inputs, done, lengths, softplus, keep)
    return y, new_state


def selective_step(u: torch.Tensor, delta: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: torch.Tensor | None,
                   state: torch.Tensor, *, z: torch.Tensor | None = None, delta_bias: torch.Tensor | None = None, softplus: bool = False,
                   reset: torch.Tensor | None = None) -> torch.Tensor:
    """``selective_scan`` for one token a row: u, delta, z (R, C), B, C (R, N) or (R, G, N) -> y (R, C).  ``state``
    (R, C, N) float32, contiguous, moves on in place; rows of ``reset`` (R,) bool start from zeros.  Forward only."""
    _forward_only("selective_step", u, delta, A, B, C, D, state, z, delta_bias)
    B, C = _grouped("selective_step", "B", B, 2), _grouped("selective_step", "C", C, 2)
    run = _capi.host if _ops.direct(u) else _sequence_ops
    return run.selective_step(u, delta, A, B, C, D, state, z, delta_bias, reset, softplus)
