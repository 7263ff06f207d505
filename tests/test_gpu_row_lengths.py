"""Lengths are clamped to 0 .. T whatever their integer type holds: values beyond 32 bits mean all steps, values below zero none."""

import pytest
import torch

from tests import test_gpu_selective as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("T", [0, 9, 300])
def test_lengths_beyond_32_bits(T):
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(T)
    given = [2 ** 63 - 1, 2 ** 32 + 5, 2 ** 31, -2 ** 32 + 3, -2 ** 63, -1, 3, T, T + 1]
    R, W, N = len(given), 12, 4
    long = torch.tensor(given, device=DEV)
    short = torch.tensor([min(max(v, 0), T) for v in given], dtype=torch.int32, device=DEV)
    w = S._r(g, W, 4).to(DEV)
    u, delta, A, B, C, D, z, bias, state = [t.to(DEV).requires_grad_(True) for t in S._scan_inputs(g, T, R, W, N, 1, torch.float32)]
    runs = []
    for lengths in (long, short):
        x, taps = bnb.causal_conv(u, w, lengths=lengths, activation="silu")
        y, st = bnb.selective_scan(x, delta, A, B, C, D, z=z, delta_bias=bias, softplus=True, state=state, lengths=lengths)
        runs.append([y, st, taps, *torch.autograd.grad([y, st, taps], [u, delta, A, B, C, state], [torch.ones_like(v) for v in (y, st, taps)])])
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    assert not runs[0][0][:, 3:6].any() and torch.equal(runs[0][1][3:6], state[3:6])
    if T:
        assert bool(runs[0][0][-1, :3].any())
