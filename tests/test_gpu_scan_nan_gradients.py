"""A NaN among a step's values is a NaN in the gradients of B and C that it enters, in every type and with every count of lanes."""

import pytest
import torch

from tests import test_gpu_selective as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", S.TYPES)
@pytest.mark.parametrize("N", [4, 8, 16, 32, 64])
@pytest.mark.parametrize("W", [40, 300])     # one tile of a group's channels, several
def test_nan_is_not_lost(dtype, N, W):
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(N)
    T, R, bad = 24, 2, 10
    u, delta, A, B, C, D, z, bias, state = [t.to(DEV) for t in S._scan_inputs(g, T, R, W, N, 1, dtype)]
    dy = S._r(g, T, R, W, dtype=dtype).to(DEV)
    for where in ("u", "dy"):
        v, gy = u.clone(), dy.clone()
        (v if where == "u" else gy)[bad, 0, 3] = float("nan")
        b, c = B.clone().requires_grad_(True), C.clone().requires_grad_(True)
        y, _ = bnb.selective_scan(v, delta, A, b, c, D, z=z, delta_bias=bias, softplus=True, state=state)
        db, dc = torch.autograd.grad(y, [b, c], gy)
        db, dc = torch.isnan(db).flatten(2), torch.isnan(dc).flatten(2)
        if where == "u":     # d B = sum g p u of the step, d C = sum dy h from there on
            assert bool(db[bad, 0].all()) and bool(dc[bad:, 0].all())
        else:                # d C of the step, and g up to there
            assert bool(dc[bad, 0].all()) and bool(db[:bad + 1, 0].all())
        assert not db[:, 1].any() and not dc[:, 1].any()     # the other row
