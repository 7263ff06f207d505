"""Calls without channels or without rows: every gradient is defined, and zero where it sums over nothing."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T,R,W,G", [(5, 3, 0, 1), (5, 3, 0, 2), (5, 0, 8, 2), (0, 3, 8, 1), (0, 0, 0, 1)])
def test_gradients_of_empty_scans(T, R, W, G):
    import boost_and_broadside_b200 as bnb

    N = 16
    z = lambda *s: torch.ones(s, device=DEV, requires_grad=True)  # noqa: E731
    u, delta, A, B, C, D, bias, state = z(T, R, W), z(T, R, W), z(W, N), z(T, R, G, N), z(T, R, G, N), z(W), z(W), z(R, W, N)
    y, st = bnb.selective_scan(u, delta, A, B, C, D, delta_bias=bias, softplus=True, state=state)
    assert y.shape == u.shape and st.shape == state.shape
    leaves = [u, delta, A, B, C, D, bias, state]
    poison = [torch.full(t.shape, float("nan"), device=DEV) for t in leaves for _ in range(2)]
    del poison           # what a gradient's memory holds before it is written
    got = torch.autograd.grad([y, st], leaves, [torch.ones_like(y), torch.ones_like(st)])
    for a, t in zip(got, leaves):
        assert a.shape == t.shape
        assert torch.equal(a, torch.ones_like(a) if t is state else torch.zeros_like(a))


@pytest.mark.parametrize("T,R,W", [(5, 3, 0), (5, 0, 8), (0, 3, 8)])
def test_gradients_of_empty_convolutions(T, R, W):
    import boost_and_broadside_b200 as bnb

    z = lambda *s: torch.ones(s, device=DEV, requires_grad=True)  # noqa: E731
    x, w, b, state = z(T, R, W), z(W, 4), z(W), z(R, 3, W)
    y, st = bnb.causal_conv(x, w, b, state=state)
    leaves = [x, w, b, state]
    poison = [torch.full(t.shape, float("nan"), device=DEV) for t in leaves for _ in range(2)]
    del poison
    got = torch.autograd.grad([y, st], leaves, [torch.ones_like(y), torch.ones_like(st)])
    for a, t in zip(got, leaves):
        assert a.shape == t.shape
        if T == 0 or R == 0 or W == 0:
            assert torch.equal(a, torch.ones_like(a) if t is state else torch.zeros_like(a))
