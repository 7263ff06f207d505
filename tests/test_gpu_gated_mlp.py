"""``gated_mlp`` against its 64-bit implementation: odd sizes, no rows, every type, strided inputs, gradients; the module that calls
it; captured and compiled calls.

Tolerances are first-order error bounds, elementwise: a result in a 16-bit type and every 16-bit operand between two
products is off by half a step e = eps / 2 of its type relative to its value; a sum over depth k on the tensor cores by
(k / 16 + 8) 2^-23 relative to the sum of its terms' sizes (one truncated addition for every sixteen products, some roundings);
the activation's value by 4e-7 (1 + |g|) and its slope by 1e-6.  |act'| <= 1.13 and |act''| <= 0.8 for both activations.
"""

import pytest
import torch

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.numel() == 0:
        return
    err = (got.detach().cpu().double() - want).abs()
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37
    bound = 1.1 * bound + tiny      # products of two errors
    assert bool((err <= bound).all()), f"{what}: off by {float((err / bound).max()):.2f} times what is allowed"


def _half(t):
    return 0.0 if t.dtype == torch.float32 else torch.finfo(t.dtype).eps / 2


def _bounds(x, wg, wu, wd, dy, act, wide_weights):
    """Values and error bounds of y, dx, dWg, dWu, dWd.  wide_weights: float32 weights of a 16-bit call, rounded to its type."""
    e = _half(x)
    s = lambda depth: (depth / 16 + 8) * 2.0 ** -23  # noqa: E731
    X, G, U, W, DY = (t.double() for t in (x, wg, wu, wd, dy))
    D, F, M = X.shape[1], G.shape[0], X.shape[0]
    g, u = X @ G.T, X @ U.T
    leaf = g.clone().requires_grad_(True)
    a = torch.nn.functional.silu(leaf) if act == "silu" else torch.nn.functional.gelu(leaf)
    da, = torch.autograd.grad(a.sum(), leaf)
    a = a.detach()
    h, dh = a * u, DY @ W
    gs, us = s(D) * (X.abs() @ G.abs().T), s(D) * (X.abs() @ U.abs().T)

    def hidden(eg, eu):
        ea = 1.13 * eg + 4e-7 * (1 + g.abs())
        return ea, u.abs() * ea + a.abs() * eu + e * h.abs()

    y = h @ W.T
    _, eh = hidden(gs, us)
    out = [(y, eh @ W.abs().T + s(F) * (h.abs() @ W.abs().T) + e * y.abs())]
    eg, eu = gs + e * g.abs(), us + e * u.abs()     # kept in x's type
    ea, eh = hidden(eg, eu)
    eda = 0.8 * eg + 1e-6
    edh = s(D) * (DY.abs() @ W.abs())
    dg, du = dh * u * da, dh * a
    edg = dh.abs() * (u.abs() * eda + da.abs() * eu) + (u * da).abs() * edh + e * dg.abs()
    edu = dh.abs() * ea + a.abs() * edh + e * du.abs()
    dx = dg @ G + du @ U
    out.append((dx, edg @ G.abs() + edu @ U.abs() + s(2 * F) * (dg.abs() @ G.abs() + du.abs() @ U.abs()) + e * dx.abs()))
    ew = 0.0 if wide_weights else e
    for left, el, right, er in ((dg, edg, X, 0.0), (du, edu, X, 0.0), (DY, 0.0, h, eh)):
        v = left.T @ right
        b = s(M) * (left.abs().T @ right.abs()) + ew * v.abs()
        if torch.is_tensor(el):
            b = b + el.T @ right.abs()
        if torch.is_tensor(er):
            b = b + left.abs().T @ er
        out.append((v, b))
    return out


CASES = [
    # rows, width, hidden, type, float32 weights, activation
    (1, 8, 8, torch.bfloat16, False, "gelu"),
    (1, 1, 1, torch.float32, False, "silu"),
    (2, 17, 5, torch.float16, True, "silu"),
    (16, 128, 512, torch.bfloat16, True, "gelu"),
    (127, 33, 100, torch.float32, False, "gelu"),
    (128, 64, 64, torch.float16, False, "gelu"),
    (129, 72, 129, torch.bfloat16, False, "silu"),
    (300, 136, 200, torch.bfloat16, True, "silu"),
    (300, 130, 257, torch.float32, False, "silu"),
    (1000, 128, 512, torch.float16, False, "gelu"),
    (2500, 96, 40, torch.bfloat16, False, "gelu"),        # weight gradients over a cut depth
    (40, 40, 2600, torch.float32, False, "gelu"),         # the down projection over a cut depth
    (200, 640, 320, torch.float16, True, "silu"),
    (20000, 24, 48, torch.bfloat16, False, "silu"),       # more tiles than SMs
]


@pytest.mark.parametrize("M,D,F,dtype,wide,act", CASES)
def test_gated_mlp(M, D, F, dtype, wide, act):
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(M + D)
    x, dy = (torch.randn(M, D, generator=g).to(dtype) for _ in range(2))
    ws = [(torch.randn(a, b, generator=g) * b ** -0.5).to(dtype) for a, b in ((F, D), (F, D), (D, F))]
    want = _bounds(x, *ws, dy, act, wide)
    leaves = [x.to(DEV).requires_grad_(True)] + [(w.float() if wide else w).to(DEV).requires_grad_(True) for w in ws]
    y = bnb.gated_mlp(*leaves, activation=act)
    assert y.dtype == dtype
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    for name, a, (v, b) in zip(("y", "dx", "d gate_w", "d up_w", "d down_w"), (y, *got), want):
        _within(a, v, b, name)
    assert all(a.dtype == t.dtype for a, t in zip(got, leaves))
    with torch.no_grad():
        assert torch.equal(bnb.gated_mlp(*leaves, activation=act), y)
    again = torch.autograd.grad(bnb.gated_mlp(*leaves, activation=act), leaves, dy.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    from boost_and_broadside_b200 import _capi
    torch.cuda.synchronize()
    assert _capi.lib.bnb_last_status() == 0


def test_layouts_and_empty_batches():
    """Leading dims, columns of a wider tensor at an odd offset, transposed weights, an expanded gradient, no rows at all."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(2)
    D, F = 40, 56
    wide = torch.randn(3, 5, D + 9, generator=g).to(torch.bfloat16).to(DEV)
    x = wide[..., 3:3 + D].requires_grad_(True)
    ws = [torch.randn(D, F, generator=g).to(DEV).t().requires_grad_(True), torch.randn(F, D, generator=g).to(DEV).requires_grad_(True),
          torch.randn(F, D, generator=g).to(DEV).t().requires_grad_(True)]
    y = bnb.gated_mlp(x, *ws)
    dense = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in (x, *ws)]
    z = bnb.gated_mlp(*dense)
    assert torch.equal(y, z)
    one = torch.ones((), dtype=torch.bfloat16, device=DEV).expand(3, 5, D)
    for a, b in zip(torch.autograd.grad(y, [x, *ws], one), torch.autograd.grad(z, dense, one.contiguous())):
        assert torch.equal(a, b)
    none = torch.zeros(0, 4, D, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    y = bnb.gated_mlp(none, *ws)
    assert y.shape == none.shape
    grads = torch.autograd.grad(y, [none, *ws], torch.zeros_like(y))
    assert grads[0].shape == none.shape and not any(v.any() for v in grads[1:])


def test_gradient_against_differences():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(3)
    M, D, F = 50, 24, 40
    ins = [torch.randn(M, D, generator=g, dtype=torch.float64)] + [torch.randn(a, b, generator=g, dtype=torch.float64) * b ** -0.5 for a, b in ((F, D), (F, D), (D, F))]
    way = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in ins]
    dy = torch.randn(M, D, generator=g, dtype=torch.float64)
    at = lambda e: float((O.gated_mlp(*[t + e * v for t, v in zip(ins, way)]) * dy).sum())  # noqa: E731
    slope = (at(1e-5) - at(-1e-5)) / 2e-5
    leaves = [t.float().to(DEV).requires_grad_(True) for t in ins]
    grads = torch.autograd.grad(bnb.gated_mlp(*leaves), leaves, dy.float().to(DEV))
    parts = [(a.double().cpu() * v) for a, v in zip(grads, way)]
    assert abs(sum(float(p.sum()) for p in parts) - slope) <= 1e-5 * sum(float(p.abs().sum()) for p in parts)


def test_module_is_differentiable_through_the_operator():
    """GatedMLP with an input that requires grad: the block's gradients, for float32 and under autocast; without, as before."""
    import boost_and_broadside_b200 as bnb

    torch.manual_seed(4)
    mlp = bnb.GatedMLP(64).to(DEV)
    x = torch.randn(7, 3, 64, device=DEV)
    for bf16 in (False, True):
        xg = x.clone().requires_grad_(True)
        with torch.autocast(DEV, dtype=torch.bfloat16, enabled=bf16):
            y = mlp(xg)
            with torch.no_grad():
                plain = mlp(x)
        assert y.dtype == plain.dtype == (torch.bfloat16 if bf16 else torch.float32) and y.shape == x.shape
        assert float((y.float() - plain.float()).abs().max()) <= (2e-2 if bf16 else 1e-5) * float(plain.float().abs().max())
        leaves = [xg, *mlp.parameters()]
        got = torch.autograd.grad(y, leaves, torch.ones_like(y))
        wl = [t.detach().cpu().double().requires_grad_(True) for t in (x, mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight)]
        want = torch.autograd.grad(O.gated_mlp(*wl), wl, torch.ones(x.shape, dtype=torch.float64))
        for a, v in zip(got, want):
            assert a.dtype == torch.float32
            assert float((a.cpu().double() - v).norm()) <= (2e-2 if bf16 else 1e-5) * float(v.norm())


def test_captured_compiled_and_second_order():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(5)
    M, D, F = 70, 64, 96
    x = torch.randn(M, D, generator=g).to(torch.bfloat16).to(DEV).requires_grad_(True)
    ws = [(torch.randn(a, b, generator=g) * b ** -0.5).to(DEV).requires_grad_(True) for a, b in ((F, D), (F, D), (D, F))]
    dy = torch.randn(M, D, generator=g).to(torch.bfloat16).to(DEV)

    def run():
        y = bnb.gated_mlp(x, *ws, activation="silu")
        return y.detach(), *torch.autograd.grad(y, [x, *ws], dy)

    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run()
    with torch.no_grad():
        x.copy_(torch.randn(M, D, generator=g))
        ws[0].mul_(1.5)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, run()))

    block = lambda x, *ws: bnb.gated_mlp(x, *ws, activation="silu")  # noqa: E731
    y = block(x, *ws)
    z = torch.compile(block, fullgraph=True)(x, *ws)
    assert torch.equal(y, z)
    for a, b in zip(torch.autograd.grad(y, [x, *ws], dy), torch.autograd.grad(z, [x, *ws], dy)):
        assert torch.equal(a, b)
    first, = torch.autograd.grad(block(x, *ws), [x], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(first.float().sum(), [ws[0]])
