"""Plain 64-bit implementations of the recurrent operators outside the trunk, step by step on the CPU (test
infrastructure only).  Differentiable by autograd; every argument is taken to float64 first."""

from __future__ import annotations

import torch
import torch.nn.functional as F


def _d(t):
    return None if t is None else t.double() if t.is_floating_point() else t


def causal_conv(x, weight, bias=None, state=None, done=None, lengths=None, activation=None):
    """x (T, R, C), weight (C, K) -> (y (T, R, C), state (R, K-1, C))."""
    x, weight, bias, state = (_d(t) for t in (x, weight, bias, state))
    T, R, C = x.shape
    K = weight.shape[1]
    taps = torch.zeros(R, K - 1, C, dtype=torch.float64) if state is None else state
    ys = []
    for t in range(T):
        live = torch.ones(R, dtype=torch.bool) if lengths is None else lengths > t
        held = taps
        if t > 0 and done is not None:
            taps = torch.where(done[t - 1][:, None, None], 0.0, taps)
        now = torch.where(live[:, None], x[t], 0.0)
        window = torch.cat([taps, now[:, None]], 1)                     # (R, K, C), oldest first
        pre = (window * weight.t()).sum(1) + (0.0 if bias is None else bias)
        y = F.silu(pre) if activation == "silu" else pre
        ys.append(torch.where(live[:, None], y, 0.0))
        taps = torch.where(live[:, None, None], window[:, 1:], held)
    return (torch.stack(ys) if ys else x), taps


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, done=None, lengths=None):
    """u, delta, z (T, R, W), A (W, N), B, C (T, R, G, N) -> (y (T, R, W), state (R, W, N))."""
    u, delta, A, B, C, D, z, delta_bias, state = (_d(t) for t in (u, delta, A, B, C, D, z, delta_bias, state))
    T, R, W = u.shape
    N, G = A.shape[1], B.shape[-2]
    h = torch.zeros(R, W, N, dtype=torch.float64) if state is None else state
    ys = []
    for t in range(T):
        live = torch.ones(R, dtype=torch.bool) if lengths is None else lengths > t
        on = live[:, None]
        held = h
        if t > 0 and done is not None:
            h = torch.where(done[t - 1][:, None, None], 0.0, h)
        ut, dt = torch.where(on, u[t], 0.0), torch.where(on, delta[t], 0.0)
        bt, ct = (torch.where(on[..., None], v[t], 0.0).repeat_interleave(W // G, 1) for v in (B, C))
        p = dt if delta_bias is None else dt + delta_bias
        p = F.softplus(p, threshold=50.0) if softplus else p
        h = torch.exp(p[..., None] * A) * h + (p * ut)[..., None] * bt
        y = (h * ct).sum(-1)
        if D is not None:
            y = y + D * ut
        if z is not None:
            y = y * F.silu(torch.where(on, z[t], 0.0))
        ys.append(torch.where(on, y, 0.0))
        h = torch.where(on[..., None], h, held)
    return (torch.stack(ys) if ys else u), h


def gated_mlp(x, gate_w, up_w, down_w, activation="gelu"):
    """down(act(gate(x)) * up(x)); act is erf GELU or SiLU."""
    x, gate_w, up_w, down_w = (_d(t) for t in (x, gate_w, up_w, down_w))
    g = x @ gate_w.t()
    return ((F.silu(g) if activation == "silu" else F.gelu(g)) * (x @ up_w.t())) @ down_w.t()
