"""Sequences of few rows are computed in splits of time, joined by the decay over a split, which may be beyond float32 where no step's
is: states that are zero stay zero, others come out as step by step.

Tolerances are those of test_gpu_selective.py.
"""

import pytest
import torch

from oracle import sequence_oracle as O
from tests import test_gpu_selective as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _against_oracle(inputs, dy, ds, done=None, close=None):
    import boost_and_broadside_b200 as bnb

    T, R, W = inputs[0].shape
    N = inputs[2].shape[1]
    wl = [None if t is None else t.double().requires_grad_(True) for t in inputs]
    wy, wst = O.selective_scan(*wl[:8], softplus=False, state=wl[8], done=done)
    given = [t for t in wl if t is not None]
    want = torch.autograd.grad([wy, wst], given, [dy.double(), ds.double()])
    assert all(bool((v.abs() < 1e37).all()) for v in (wy, wst, *want))     # float32 holds them
    leaves = [None if t is None else t.to(DEV).requires_grad_(True) for t in inputs]
    u, delta, A, B, C, D, z, bias, state = leaves
    y, st = bnb.selective_scan(u, delta, A, B, C, D, z=z, delta_bias=bias, state=state, done=S._dev(done)[0])
    got = torch.autograd.grad([y, st], [t for t in leaves if t is not None], [dy.to(DEV), ds.to(DEV)])
    S.CALL_IS_16[0] = False
    sy, sst, *sizes = S._scan_sizes(*inputs, False, done, None, dy, ds)
    S._close(y, wy, sy, T, N, what="y")
    S._close(st, wst, sst, T, what="state")
    if close:
        assert bool(((st.detach().cpu().double() - wst.detach()).abs() <= close * wst.detach().abs()).all())
    names, terms = ["u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"], [N, N, T * R, W, W, T * R, N, T * R * N, 1]
    for (name, n, sz), a, v in zip([(m, k, q) for m, k, q, t in zip(names, terms, sizes, leaves) if t is not None], got, want):
        S._close(a, v, sz, 2 * T, n, what="d " + name)


def _growing(T, R, W, N, rate, seed):
    g = torch.Generator().manual_seed(seed)
    inputs = list(S._scan_inputs(g, T, R, W, N, 1, torch.float32))
    inputs[1] = torch.full((T, R, W), 2.0)
    inputs[2] = torch.full((W, N), rate)
    inputs[6] = inputs[7] = inputs[8] = None
    return g, inputs


@pytest.mark.parametrize("T,R,W,N", [(400, 1, 8, 4), (700, 2, 40, 16)])
def test_zero_states_stay_zero_while_they_could_grow(T, R, W, N):
    """A step's growth of e^2 is within float32, a split's of e^160 is not; inputs come at the last steps and gradients at the first alone."""
    g, inputs = _growing(T, R, W, N, 1.0, 1)
    inputs[0][: T - 3] = 0.0
    dy = torch.zeros(T, R, W)
    dy[:3] = S._r(g, 3, R, W)
    _against_oracle(inputs, dy, torch.zeros(R, W, N))


# A state alone: its decays' exponents, up to 173 as powers of two and sums of sizes that float32 holds exactly, err by 2^-24 for the constant
# log2(e) and by as much for the product, so the state by 173 ln(2) 2^-23 of itself, and two exponentials by 2^-22 each: 2e-5.
CLOSE = 2e-5


def test_small_states_grow_within_range():
    """From 1e-30 by e^100 in a split, then steps of no size."""
    T, R, W, N = 400, 1, 8, 4
    g, inputs = _growing(T, R, W, N, 1.0, 2)
    inputs[1] = torch.zeros(T, R, W)
    inputs[1][:64] = 100.0 / 64
    inputs[0][:] = 0.0
    inputs[8] = 1e-30 * (1.0 + torch.rand(R, W, N, generator=g))
    _against_oracle(inputs, 1e-20 * S._r(g, T, R, W), torch.zeros(R, W, N), close=CLOSE)


def test_large_states_decay_within_range():
    """From 1e30 by e^-120 in a split."""
    T, R, W, N = 400, 1, 8, 4
    g, inputs = _growing(T, R, W, N, -1.0, 3)
    inputs[1] = torch.zeros(T, R, W)
    inputs[1][:64] = 120.0 / 64
    inputs[0][:] = 0.0
    inputs[8] = 1e30 * (1.0 + torch.rand(R, W, N, generator=g))
    dy = torch.zeros(T, R, W)
    dy[-1] = S._r(g, R, W)
    _against_oracle(inputs, dy, torch.zeros(R, W, N), close=CLOSE)


def test_an_infinite_state_stays_infinite():
    import boost_and_broadside_b200 as bnb

    T, R, W, N = 400, 1, 8, 4
    _, inputs = _growing(T, R, W, N, -1.0, 4)
    state = torch.ones(R, W, N)
    state[0, 3, 1] = float("inf")
    args = S._dev(*inputs[:5])
    _, st = bnb.selective_scan(*args, state=state.to(DEV))
    assert float(st[0, 3, 1]) == float("inf") and int(torch.isfinite(st).sum()) == W * N - 1
