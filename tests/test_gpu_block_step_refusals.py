"""``SelectiveTemporalBlock`` refuses what it cannot compute before it moves any state on."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _states(block, R):
    g = torch.Generator().manual_seed(R)
    return [torch.randn(t.shape, generator=g).to(DEV) for t in block.initial_state(R)]


def _block():
    import boost_and_broadside_b200 as bnb

    torch.manual_seed(0)
    return bnb.SelectiveTemporalBlock(32, d_state=4).to(DEV)


def test_float16_autocast_is_refused_at_the_start():
    block, x = _block(), torch.randn(3, 32, device=DEV)
    h, taps = _states(block, 3)
    before = h.clone(), taps.clone()
    with torch.autocast(DEV, dtype=torch.float16):
        with pytest.raises(RuntimeError, match="autocast dtype"):
            block.step(x, h, taps)
        with pytest.raises(RuntimeError, match="autocast dtype"):
            block.forward_sequence(x[:, None], h, taps)
    assert torch.equal(h, before[0]) and torch.equal(taps, before[1])
    block.step(x, h, taps)
    assert not torch.equal(h, before[0])


def _misplaced(t):
    """The same values 4 bytes behind a boundary of 16."""
    wide = torch.empty(t.numel() + 1, device=DEV)
    wide[1:] = t.flatten()
    return wide[1:].view(t.shape)


@pytest.mark.parametrize("which", ["h", "conv_buf"])
@pytest.mark.parametrize("how", ["type", "strides", "boundary"])
def test_unsuitable_states_are_refused_at_the_start(which, how):
    block, x = _block(), torch.randn(3, 32, device=DEV)
    states = dict(zip(("h", "conv_buf"), _states(block, 3)))
    t = states[which]
    states[which] = t.half() if how == "type" else _misplaced(t) if how == "boundary" else t.transpose(1, 2).contiguous().transpose(1, 2)
    before = {k: v.clone() for k, v in states.items()}
    with pytest.raises(RuntimeError):
        block.step(x, **states)
    assert all(torch.equal(states[k], before[k]) for k in states)


def test_an_unsuitable_reset_is_refused_at_the_start():
    block, x = _block(), torch.randn(3, 32, device=DEV)
    h, taps = _states(block, 3)
    before = h.clone(), taps.clone()
    with pytest.raises(RuntimeError, match="reset"):
        block.step(x, h, taps, torch.zeros(2, dtype=torch.bool, device=DEV))
    assert torch.equal(h, before[0]) and torch.equal(taps, before[1])


def test_compiled_steps_still_run():
    block, x = _block(), torch.randn(3, 32, device=DEV)
    h, taps = _states(block, 3)
    other = h.clone(), taps.clone()
    want = block.step(x, *other)
    got = torch.compile(block.step, fullgraph=True)(x, h, taps)
    assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())
    assert float((h - other[0]).abs().max()) <= 1e-5 * float(h.abs().max()) and float((taps - other[1]).abs().max()) <= 1e-5 * float(taps.abs().max())
