"""Rows of the gated block that share memory (a gradient expanded from one row, a broadcast input): the products' operands are described by
strides that do not overlap, so such rows are copied first."""

import ctypes as C

import pytest
import torch

from tests.test_sequence_refusals import Gated

DEV = "cuda"


@pytest.mark.parametrize("element", [1, 2])
def test_rows_closer_than_their_width_count_as_copied(element):
    from boost_and_broadside_b200 import _capi

    fake = 0x1000

    def need(x_row):
        c = Gated(100, 64, 128, element, element, 2, fake, x_row, fake, fake, fake, fake, None)
        return _capi.lib.bnb_gated_block_scratch_bytes(C.byref(c), 0)

    copy = 100 * 64 * 2 + (-100 * 64 * 2) % 256
    assert need(72) == need(64) and need(65) == need(64) + copy      # as they lie; off a boundary of 16 bytes
    assert need(0) == need(56) == need(8) == need(64) + copy


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,D,F", [(5, 40, 56), (300, 64, 128)])
def test_expanded_rows(dtype, M, D, F):
    """A sum over rows hands every row the same gradient, one that lies in memory once."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(M)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    x, ws, dy = r(M, D), [r(F, D), r(F, D), r(D, F)], r(D)
    leaves = [t.requires_grad_(True) for t in (x, *ws)]
    got = torch.autograd.grad(bnb.gated_mlp(*leaves), leaves, dy.expand(M, D))
    want = torch.autograd.grad(bnb.gated_mlp(*leaves), leaves, dy.expand(M, D).contiguous())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = torch.autograd.grad((bnb.gated_mlp(*leaves).sum(0) * dy).sum(), leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = x.detach()[:1].expand(M, D)
    assert torch.equal(bnb.gated_mlp(one, *ws), bnb.gated_mlp(one.contiguous(), *ws))
    overlapping = r(M * 8 + D).as_strided((M, D), (8, 1))
    assert torch.equal(bnb.gated_mlp(overlapping, *ws), bnb.gated_mlp(overlapping.contiguous(), *ws))
