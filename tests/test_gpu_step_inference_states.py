"""States made in inference mode: single tokens move them on in that mode, and outside of it refuse before they do."""

import pytest
import torch

from tests import test_gpu_selective as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("name", ["conv", "scan", "block"])
def test_states_of_inference_mode(name):
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(1)
    R, W, N = 3, 8, 4
    u, delta, A, B, C, D, z, bias, _ = [t.to(DEV) for t in S._scan_inputs(g, 1, R, W, N, 1, torch.float32)]
    w = S._r(g, W, 4).to(DEV)
    torch.manual_seed(0)
    block = bnb.SelectiveTemporalBlock(W // 2, d_state=N).to(DEV)
    taps, h = S._r(g, R, 3, W), S._r(g, R, W, N)

    def call(taps, h):
        if name == "conv":
            return bnb.causal_conv_step(u[0], taps, w)
        if name == "scan":
            return bnb.selective_step(u[0], delta[0], A, B[0], C[0], D, h, softplus=True)
        return block.step(u[0, :, : W // 2], h, taps)

    plain = taps.to(DEV), h.to(DEV)
    with torch.no_grad():
        want = call(*plain)
    with torch.inference_mode():
        held = taps.to(DEV), h.to(DEV)
    before = [t.clone() for t in held]
    for states in (held, (plain[0].clone(), held[1]), (held[0], plain[1].clone())) if name == "block" else (held,):
        kept = [t.clone() for t in states]
        with torch.no_grad(), pytest.raises(RuntimeError, match="inference"):
            call(*states)
        assert all(torch.equal(a, b) for a, b in zip(states, kept))
    with torch.inference_mode():
        got = call(*held)
        assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(held, plain))
    assert not all(torch.equal(a, b) for a, b in zip(held, before))
