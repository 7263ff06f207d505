"""Step sizes masked by -inf or by a type's lowest value: softplus is 0 there, so the step leaves the state alone, in sequences, their
gradients and single tokens; a step of infinite size and a step that is no number stay what they are.

Tolerances are those of test_gpu_selective.py.
"""

import pytest
import torch

from oracle import sequence_oracle as O
from tests import test_gpu_selective as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(T, R, W, N, dtype, fill, seed):
    """The first half of a row's steps and every third one behind are masked."""
    g = torch.Generator().manual_seed(seed)
    inputs = list(S._scan_inputs(g, T, R, W, N, 1, dtype))
    masked = (torch.arange(T) < T // 2) | (torch.arange(T) % 3 == 0)
    inputs[1][masked] = -float("inf") if fill == "-inf" else torch.finfo(dtype).min
    return g, inputs, masked


@pytest.mark.parametrize("T,R,W,N", [(24, 3, 10, 16), (400, 1, 8, 4), (19, 2, 33, 64)])   # the second: several splits of time
@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("fill", ["-inf", "lowest"])
def test_masked_steps_leave_the_state_alone(T, R, W, N, dtype, fill):
    import boost_and_broadside_b200 as bnb

    g, inputs, _ = _inputs(T, R, W, N, dtype, fill, T + N)
    dy, ds = S._r(g, T, R, W, dtype=dtype), S._r(g, R, W, N)
    wl = [t.double().requires_grad_(True) for t in inputs]
    wy, wst = O.selective_scan(*wl[:8], softplus=True, state=wl[8])
    want = torch.autograd.grad([wy, wst], wl, [dy.double(), ds.double()])
    assert all(bool(torch.isfinite(v).all()) for v in (wy, wst, *want))

    leaves = [t.to(DEV).requires_grad_(True) for t in inputs]
    u, delta, A, B, C, D, z, bias, state = leaves
    y, st = bnb.selective_scan(u, delta, A, B, C, D, z=z, delta_bias=bias, softplus=True, state=state)
    got = torch.autograd.grad([y, st], leaves, [dy.to(DEV), ds.to(DEV)])
    S.CALL_IS_16[0] = dtype != torch.float32
    lowered = [t.clamp(min=-1e4) if i == 1 else t for i, t in enumerate(inputs)]   # the same step sizes of 0, and no inf * 0 among the sizes
    sy, sst, *sizes = S._scan_sizes(*lowered, True, None, None, dy, ds)
    S._close(y, wy, sy, T, N, what="y")
    S._close(st, wst, sst, T, what="state")
    terms = [N, N, T * R, W, W, T * R, N, T * R * N, 1]
    for name, a, v, sz, n in zip(("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"), got, want, sizes, terms):
        S._close(a, v, sz, 2 * T, n, what="d " + name)


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("N", [16, 6, 64])
def test_a_masked_token_leaves_the_state_alone(dtype, N):
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(N)
    R, W = 6, 36
    u, delta, A, B, C, D, z, bias, state = [t.to(DEV) for t in S._scan_inputs(g, 1, R, W, N, 1, dtype)]
    delta = delta.clone()
    delta[0, 0] = -float("inf")
    delta[0, 1] = torch.finfo(dtype).min
    held = state.clone()
    y = bnb.selective_step(u[0], delta[0], A, B[0], C[0], D, held, z=z[0], delta_bias=bias, softplus=True)
    assert torch.equal(held[:2], state[:2]) and bool(torch.isfinite(y).all()) and bool(torch.isfinite(held).all())
    assert not torch.equal(held[2:], state[2:])


def test_infinite_steps_and_no_numbers_stay():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(3)
    T, R, W, N = 9, 2, 8, 4
    u, delta, A, B, C, D, z, bias, state = S._scan_inputs(g, T, R, W, N, 1, torch.float32)
    delta[T - 1, 0, 2] = float("inf")
    delta[4, 1, 5] = float("nan")
    wy, wst = O.selective_scan(u, delta, A, B, C, D, z, None, True, state)
    y, st = bnb.selective_scan(*S._dev(u, delta, A, B, C, D), z=z.to(DEV), softplus=True, state=state.to(DEV))
    held = state.to(DEV)
    for t in range(T):
        last = bnb.selective_step(*S._dev(u[t], delta[t], A, B[t], C[t], D), held, z=z[t].to(DEV), softplus=True)
    inf = float("inf")
    assert bool((wst[0, 2].abs() == inf).all()) and bool(torch.isnan(wst[1, 5]).all())
    for got in (st.cpu().double(), held.cpu().double()):
        assert torch.equal(got[0, 2], wst[0, 2]) and bool(torch.isnan(got[1, 5]).all())
    for got, want in ((y.cpu().double(), wy), (last.cpu().double(), wy[T - 1])):
        assert torch.equal(torch.isfinite(got), torch.isfinite(want))
