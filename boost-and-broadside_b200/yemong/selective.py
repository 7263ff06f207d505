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
once on the way out; the terms of the sums over channels that are the gradients of B and C enter them with 16 bits
(bfloat16) or 22 (others), up to 32 states.  Decays and step sizes are good to a few units of 2^-23 in every type.
"""

from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import _capi
from . import _ops, _sequence_ops
from ._sequence_ops import activation_code
from .attention import GatedMLP
from .gated import gated_mlp

TAPS: int = 4  # of the block's convolution, as CONV_KERNEL of the Griffin sublayer (griffin.py:22)


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

    A step is masked by delta = -inf or its type's lowest value where ``softplus`` is asked for: its size is 0, the state stays.

    An infinity or NaN among an episode's values stays in it, with one exception: the gradients of B and C may show it in
    the row's other episodes too, up to eight steps away.  An infinity may come out as NaN: in those gradients, and in y
    where N is not 4, 8, 16, 32 or 64.
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


class SelectiveTemporalBlock(nn.Module):
    """A temporal sublayer on these operators, in the place and with the signatures of ``GriffinTemporalBlock``
    (griffin.py:222-286).  Projections, parameters' names and starting values are those of the selective state space layer that
    Gu and Dao published (2023, arXiv:2312.00752), inside that sublayer's frame: norm -> in_proj -> (causal conv -> selective scan) gated -> out_proj -> residual
    -> gated feed-forward (norm) -> residual, per row across time.

    Its state is wider than the Griffin sublayer's: (R, E, N) and the taps (R, 3, E), E = expand * d_model channels of N
    states, whose decay depends on the input.  Whole sequences are differentiable; ``step`` moves the state on in
    place for rollouts.  Any d_model; float32, or bfloat16 activations inside ``torch.autocast``.

    Args:
        d_model: width of the tokens.
        d_state: N, states a channel (1 to 64).
        expand: E / d_model.
        dt_rank: rank of the step sizes' projection, d_model / 16 rounded up by default.
    """

    def __init__(self, d_model: int, d_state: int = 16, expand: int = 2, dt_rank: int | None = None) -> None:
        super().__init__()
        if not 1 <= d_state <= 64:
            raise ValueError(f"d_state must be between 1 and 64, got {d_state}")
        E = expand * d_model
        self.d_model, self.d_state, self.d_inner = d_model, d_state, E
        self.dt_rank = (d_model + 15) // 16 if dt_rank is None else dt_rank
        self.norm1 = nn.RMSNorm(d_model)
        self.in_proj = nn.Linear(d_model, 2 * E, bias=False)
        self.conv = nn.Conv1d(E, E, kernel_size=TAPS, groups=E, bias=True)
        self.x_proj = nn.Linear(E, self.dt_rank + 2 * d_state, bias=False)
        self.dt_proj = nn.Linear(self.dt_rank, E, bias=True)
        self.A_log = nn.Parameter(torch.log(torch.arange(1, d_state + 1, dtype=torch.float32)).repeat(E, 1))
        self.D = nn.Parameter(torch.ones(E))
        self.out_proj = nn.Linear(E, d_model, bias=False)
        self.norm2 = nn.RMSNorm(d_model)
        self.gated_mlp = GatedMLP(d_model)
        with torch.no_grad():   # step sizes of 0.001 to 0.1 at a zero input
            rate = torch.exp(torch.rand(E) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
            self.dt_proj.bias.copy_(rate + torch.log(-torch.expm1(-rate)))

    def initial_state(self, rows: int, device=None) -> tuple[torch.Tensor, torch.Tensor]:
        """(h (R, E, N), conv_buf (R, 3, E)), zeros."""
        return (torch.zeros(rows, self.d_inner, self.d_state, device=device), torch.zeros(rows, TAPS - 1, self.d_inner, device=device))

    def _projected(self, u: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """delta, B and C of the conv's output."""
        dt, B, C = self.x_proj(u).split([self.dt_rank, self.d_state, self.d_state], dim=-1)
        return F.linear(dt, self.dt_proj.weight), B, C

    def _feed_forward(self, x: torch.Tensor) -> torch.Tensor:
        mlp, n = self.gated_mlp, self.norm2(x)
        if _capi.current_precision(x.device) == _capi.BNB_BF16:
            n = n.to(torch.bfloat16)
        return x + gated_mlp(n, mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight).to(x.dtype)

    def _check(self, x: torch.Tensor, dims: int, h: torch.Tensor, conv_buf: torch.Tensor) -> None:
        if x.dim() != dims or x.shape[-1] != self.d_model:
            raise RuntimeError(f"expected an input of {dims} dims ending in {self.d_model}, got {tuple(x.shape)}")
        R = x.shape[0]
        if tuple(h.shape) != (R, self.d_inner, self.d_state) or tuple(conv_buf.shape) != (R, TAPS - 1, self.d_inner):
            raise RuntimeError("h / conv_buf shapes do not match the input")
        _capi.require_cuda(x, "x")
        _capi.current_precision(x.device)   # refuses what the feed-forward half would refuse behind the state's update

    def _check_in_place(self, x: torch.Tensor, **states: torch.Tensor) -> None:
        """What the operators ask of a state that they move on, of both before either is."""
        for name, t in states.items():
            if t.device != x.device or t.dtype != torch.float32:
                raise RuntimeError(f"{name} must be float32 on the input's device {x.device}, got {t.dtype} on {t.device}")
            if not t.is_contiguous():
                raise RuntimeError(f"{name} is updated in place and must be contiguous")
            if not _ops.direct(t):   # what cannot be traced the operators ask themselves
                continue
            if t.data_ptr() % 16:
                raise RuntimeError(f"{name} is updated in place and must lie on a 16-byte boundary")
            if t.is_inference() and not torch.is_inference_mode_enabled():
                raise RuntimeError(f"{name} is updated in place and was made in inference mode, outside of which it must not be changed")

    def forward_sequence(
        self,
        x_seq: torch.Tensor,  # (R, T, D)
        h0: torch.Tensor,  # (R, E, N)
        conv_buf: torch.Tensor,  # (R, 3, E)
        done_mask: torch.Tensor | None = None,  # (R, T) bool
        lengths: torch.Tensor | None = None,  # (R,) int
    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Returns (out (R, T, D), new_h (R, E, N), new_conv_buf (R, 3, E)).  Outputs behind a row's length are those of the
        feed-forward half alone."""
        self._check(x_seq, 3, h0, conv_buf)
        x = x_seq.transpose(0, 1)   # time-major, as it lies
        done = None if done_mask is None else done_mask.transpose(0, 1)
        u, z = self.in_proj(self.norm1(x)).split(self.d_inner, dim=-1)
        u, taps = causal_conv(u, self.conv.weight[:, 0], self.conv.bias, state=conv_buf, done=done, lengths=lengths, activation="silu")
        delta, B, C = self._projected(u)
        y, h = selective_scan(u, delta, -torch.exp(self.A_log), B, C, self.D, z=z, delta_bias=self.dt_proj.bias, softplus=True,
                              state=h0, done=done, lengths=lengths)
        return self._feed_forward(x + self.out_proj(y).to(x.dtype)).transpose(0, 1), h, taps

    @torch.no_grad()
    def step(self, x: torch.Tensor, h: torch.Tensor, conv_buf: torch.Tensor, reset: torch.Tensor | None = None) -> torch.Tensor:
        """One token a row, without gradients: x (R, D) -> (R, D).  ``h`` (R, E, N) and ``conv_buf`` (R, 3, E) move on in
        place; rows of ``reset`` (R,) bool start from zeros.  A call that is refused leaves both as they were."""
        self._check(x, 2, h, conv_buf)
        self._check_in_place(x, h=h, conv_buf=conv_buf)
        u, z = self.in_proj(self.norm1(x)).split(self.d_inner, dim=-1)
        u = causal_conv_step(u, conv_buf, self.conv.weight[:, 0], self.conv.bias, reset=reset, activation="silu")
        delta, B, C = self._projected(u)
        y = selective_step(u, delta, -torch.exp(self.A_log), B, C, self.D, h, z=z, delta_bias=self.dt_proj.bias, softplus=True, reset=reset)
        return self._feed_forward(x + self.out_proj(y).to(x.dtype))
