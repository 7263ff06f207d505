"""``gated_mlp`` at the sizes that take its wide product tiles, several of them a CTA, and depths in parts, against 64 bits on the device.

Tolerances are first-order bounds as in test_gpu_gated_mlp.py, and closer in one place: the gradients take g and u as the products left
them, in float32, so that no rounding to x's type enters there, only those of h, dg and du.  Those are off by half a step e relative to
their values, and by 2^-25, half a step of float16's subnormal numbers, where they are smaller than its normal ones.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _bounds(x, wg, wu, wd, dy, act, wide_weights):
    """Values and error bounds of y, dx, dWg, dWu, dWd, all on the inputs' device."""
    e = 0.0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    low = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    s = lambda depth: (depth / 16 + 8) * 2.0 ** -23  # noqa: E731
    X, G, U, W, DY = (t.double() for t in (x, wg, wu, wd, dy))
    (M, D), F = X.shape, G.shape[0]
    g, u = X @ G.T, X @ U.T
    leaf = g.clone().requires_grad_(True)
    a = torch.nn.functional.silu(leaf) if act == "silu" else torch.nn.functional.gelu(leaf)
    da, = torch.autograd.grad(a.sum(), leaf)
    a = a.detach()
    h, dh = a * u, DY @ W
    eg, eu = s(D) * (X.abs() @ G.abs().T), s(D) * (X.abs() @ U.abs().T)
    ea, eda = 1.13 * eg + 4e-7 * (1 + g.abs()), 0.8 * eg + 1e-6
    eh = u.abs() * ea + a.abs() * eu + e * h.abs() + low
    edh = s(D) * (DY.abs() @ W.abs())
    dg, du = dh * u * da, dh * a
    edg = dh.abs() * (u.abs() * eda + da.abs() * eu) + (u * da).abs() * edh + e * dg.abs() + low
    edu = dh.abs() * ea + a.abs() * edh + e * du.abs() + low
    y, dx = h @ W.T, dg @ G + du @ U
    out = [(y, eh @ W.abs().T + s(F) * (h.abs() @ W.abs().T) + e * y.abs()),
           (dx, edg @ G.abs() + edu @ U.abs() + s(2 * F) * (dg.abs() @ G.abs() + du.abs() @ U.abs()) + e * dx.abs())]
    ew = 0.0 if wide_weights else e
    for left, el, right, er in ((dg, edg, X, None), (du, edu, X, None), (DY, None, h, eh)):
        v = left.T @ right
        b = s(M) * (left.abs().T @ right.abs()) + ew * v.abs()
        b = b + (left.abs().T @ er if el is None else el.T @ right.abs())
        out.append((v, b))
    return out


def _check(M, D, F, dtype, wide, act):
    import boost_and_broadside_b200 as bnb
    from boost_and_broadside_b200 import _capi

    g = torch.Generator(DEV).manual_seed(M + D)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, dy = r(M, D).to(dtype), r(M, D).to(dtype)
    ws = [(r(a, b) * b ** -0.5).to(dtype) for a, b in ((F, D), (F, D), (D, F))]
    leaves = [x.clone().requires_grad_(True)] + [(w.float() if wide else w.clone()).requires_grad_(True) for w in ws]
    y = bnb.gated_mlp(*leaves, activation=act)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    for name, v, (want, bound) in zip(("y", "dx", "d gate_w", "d up_w", "d down_w"), got, _bounds(x, *ws, dy, act, wide)):
        off = ((v.detach().double() - want).abs() / (1.1 * bound + (2.0 ** -25 if v.dtype == torch.float16 else 1e-37))).max()
        assert float(off) <= 1, f"{name}: off by {float(off):.2f} times what is allowed"
    with torch.no_grad():
        assert torch.equal(bnb.gated_mlp(*leaves, activation=act), y)
    again = torch.autograd.grad(bnb.gated_mlp(*leaves, activation=act), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], again))
    torch.cuda.synchronize()
    assert _capi.lib.bnb_last_status() == 0


# What a product takes: 128 x the width, by how many tiles or in how many parts of the depth.
@pytest.mark.parametrize("M,D,F,dtype,wide,act", [
    (600, 1024, 2048, torch.bfloat16, False, "gelu"),      # y 128 in 3 parts, g and u kept 128, dx 256 in 7, dWg and dWu 256, dWd 128
    (2050, 1020, 2044, torch.float16, False, "silu"),      # off boundaries; y 128, g and u kept 256, dx 256 in 2
    (3000, 1100, 2500, torch.bfloat16, True, "silu"),      # every one 256 and whole, up to 4 tiles a CTA
    (1500, 600, 5000, torch.bfloat16, False, "gelu"),      # y 256 in 4 parts
    (20000, 520, 300, torch.float16, True, "gelu"),        # dWg and dWu 256 in 8 parts, dWd in 14
    (20000, 128, 512, torch.bfloat16, False, "silu"),      # g and u once more, 9 tiles a CTA; dWg and dWu 128 in parts
    (1, 1024, 4096, torch.bfloat16, False, "gelu"),        # one row of a wide layer
    (7, 2000, 999, torch.float16, False, "silu"),
])
def test_16_bits(M, D, F, dtype, wide, act):
    _check(M, D, F, dtype, wide, act)


@pytest.mark.parametrize("M,D,F,act", [(1000, 400, 1500, "gelu"), (4000, 300, 1000, "silu"), (3, 1000, 2000, "gelu")])
def test_float32(M, D, F, act):
    _check(M, D, F, torch.float32, False, act)


@pytest.mark.parametrize("M,D,F,dtype", [(1, 8, 8, torch.bfloat16), (129, 72, 129, torch.bfloat16), (1000, 128, 512, torch.float16),
                                         (300, 640, 320, torch.bfloat16)])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_gradients_take_unrounded_projections(M, D, F, dtype, act):
    """Narrow tiles to the closer bounds: recomputed g and u, and kept ones."""
    _check(M, D, F, dtype, False, act)
