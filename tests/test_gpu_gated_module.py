"""``GatedMLP`` on its own is differentiable in its weights whether or not its input requires a gradient."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("frozen", [(), ("gate_proj", "up_proj"), ("down_proj",)])
def test_weights_have_gradients_for_plain_inputs(bf16, frozen):
    import boost_and_broadside_b200 as bnb

    torch.manual_seed(4)
    mlp = bnb.GatedMLP(64).to(DEV)
    for name in frozen:
        getattr(mlp, name).weight.requires_grad_(False)
    wanted = [p for p in mlp.parameters() if p.requires_grad]
    x = torch.randn(7, 3, 64, device=DEV)
    grads = []
    for x_wants in (False, True):
        leaf = x.clone().requires_grad_(x_wants)
        with torch.autocast(DEV, dtype=torch.bfloat16, enabled=bf16):
            y = mlp(leaf)
        assert y.requires_grad and y.dtype == (torch.bfloat16 if bf16 else torch.float32)
        grads.append([y, *torch.autograd.grad(y, wanted, torch.ones_like(y))])
    assert len(grads[0]) == 4 - len(frozen) and all(torch.equal(a, b) for a, b in zip(*grads))


def test_without_anything_to_differentiate_nothing_is_recorded():
    import boost_and_broadside_b200 as bnb

    mlp = bnb.GatedMLP(64).to(DEV)
    x = torch.randn(5, 64, device=DEV)
    with torch.no_grad():
        want = mlp(x)
    assert not want.requires_grad
    got = mlp.requires_grad_(False)(x)
    assert not got.requires_grad and torch.equal(got, want)
