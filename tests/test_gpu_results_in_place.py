"""Results of differentiated calls may be changed in place, as every operator's may, whatever the layout of the inputs; they lie in memory
as the inputs do."""

import pytest
import torch

from tests import test_gpu_selective as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _calls():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(1)
    T, R, W, N = 6, 5, 24, 8
    w = S._r(g, W, 4).to(DEV)
    u, delta, A, B, C, D, z, bias, state = S._scan_inputs(g, T, R, W, N, 1, torch.float32)
    rest = [t.to(DEV) for t in (delta, A, B, C, D)]
    gate = [S._r(g, 2 * W, W).to(DEV), S._r(g, 2 * W, W).to(DEV), S._r(g, W, 2 * W).to(DEV)]
    return u, {"conv": lambda x: bnb.causal_conv(x, w, activation="silu"), "scan": lambda x: bnb.selective_scan(x, *rest, softplus=True),
               "gated": lambda x: (bnb.gated_mlp(x, *gate),)}


@pytest.mark.parametrize("layout", ["dense", "batch"])
@pytest.mark.parametrize("name", ["conv", "scan", "gated"])
@pytest.mark.parametrize("compiled", [False, True])
def test_in_place(layout, name, compiled):
    u, calls = _calls()
    fn = torch.compile(calls[name], fullgraph=True) if compiled else calls[name]
    grads = []
    for in_place in (False, True):
        x = S._layout(u, layout).requires_grad_(True)
        out = fn(x)
        if name != "gated":
            assert out[0].stride() == x.stride()
        if in_place:
            for t in out:
                t += 0.5
                torch.relu_(t)
        else:
            out = [torch.relu(t + 0.5) for t in out]
        grads.append([*out, *torch.autograd.grad(list(out), [x], [torch.full_like(t, 2.0) for t in out])])
        assert grads[-1][-1].shape == x.shape
    assert all(torch.equal(a, b) for a, b in zip(*grads))
