"""``linear`` against its 64-bit implementation: odd sizes, no rows, every type, strided inputs, gradients, the sums of a cut depth; captured and
compiled calls.

Tolerances are first-order error bounds, elementwise: a result in a 16-bit type, and the gradient before the activation as an operand, is off by
half a step e = eps / 2 of its type relative to its value; a sum over depth k on the tensor cores by (k / 16 + 8) 2^-23 relative to the sum of its
terms' sizes (one truncated addition for every sixteen products, some roundings); the activation's value by 4e-7 (1 + |z|) and its slope by
1e-6.  |act'| <= 1.13 and |act''| <= 0.8 for both activations.  A column is summed in runs of rows / 32 at most and some 100 sums of those."""

import pytest
import torch

from oracle import update_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.numel() == 0:
        return
    err = (got.detach().cpu().double() - want).abs()
    own = 0.0 if got.dtype == F32 else torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == F16 else 1e-37
    bound = 1.1 * (bound + own * want.abs()) + tiny
    assert bool((err <= bound).all()), f"{what}: off by {float((err / bound).max()):.2f} times what is allowed"


def _bounds(x, w, b, r, dy, act):
    """Values and error bounds (without their own type's rounding) of y, dx, dW, db."""
    e = 2.0 ** -24 if x.dtype == F32 else torch.finfo(x.dtype).eps / 2
    small = 2.0 ** -25 if x.dtype == F16 else 0.0     # half the least step of an operand
    s = lambda depth: (depth / 16 + 8) * 2.0 ** -23  # noqa: E731
    (M, K), N = x.shape, w.shape[0]
    X, W, DY = x.double(), w.double(), dy.double()
    z = X @ W.T + (0 if b is None else b.double())
    ez = s(K) * (X.abs() @ W.abs().T) + 2.0 ** -23 * z.abs()
    leaf = z.clone().requires_grad_(True)
    a = {None: lambda v: v * 1.0, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[act](leaf)
    da, = torch.autograd.grad(a.sum(), leaf)
    y = O.linear(x, w, b, act, r)
    ey = ez if act is None else 1.13 * ez + 4e-7 * (1 + z.abs())
    ey = ey + 2.0 ** -23 * (a.detach().abs() + y.abs())
    dz = DY * da
    wide = torch.zeros_like(dz) if act is None else DY.abs() * (0.8 * ez + 1e-6) + 2.0 ** -23 * dz.abs()     # before it is rounded as an operand
    edz = wide if act is None else wide + e * dz.abs() + small
    return [(y, ey), (dz @ W, edz @ W.abs() + s(N) * (dz.abs() @ W.abs())), (dz.T @ X, edz.T @ X.abs() + s(M) * (dz.abs().T @ X.abs())),
            (dz.sum(0), wide.sum(0) + (M / 32 + 100) * 2.0 ** -24 * dz.abs().sum(0))]


CASES = [
    # rows, width, outputs, type, float32 weight, float32 bias (None: no bias), activation, residual
    (1, 1, 1, F32, False, False, None, False),
    (1, 8, 8, BF16, False, False, "gelu", True),
    (2, 17, 5, F16, True, True, "silu", True),
    (16, 128, 256, BF16, True, True, "gelu", False),
    (16, 128, 256, F32, False, None, "gelu", True),
    (127, 33, 100, F32, False, False, "silu", True),
    (128, 64, 64, F16, False, False, None, True),
    (129, 72, 129, BF16, False, True, "silu", False),
    (300, 130, 257, F32, False, False, None, False),
    (301, 522, 130, F32, False, False, "silu", True),
    (300, 513, 200, BF16, False, False, "gelu", True),       # wide, slopes kept
    (200, 640, 321, F16, True, None, "silu", False),
    (200, 512, 64, BF16, False, False, "silu", True),        # narrow
    (2500, 96, 40, BF16, False, False, "gelu", True),        # the weight's gradient over a cut depth
    (5, 4096, 100, BF16, False, False, "gelu", True),        # a cut depth, slopes kept by its sums
    (3, 4096, 4096, F16, False, False, None, True),
    (40, 2600, 70, F32, False, False, "gelu", True),
    (1, 4100, 33, F32, False, True, "silu", False),
    (20000, 24, 48, BF16, False, False, "silu", True),       # more tiles than SMs
    (3000, 1030, 520, F16, False, False, "gelu", True),
    (1, 1024, 7, F32, False, False, "gelu", True),           # few rows
    (2, 1032, 5, F16, False, True, None, True),
    (4, 2048, 33, BF16, True, True, "silu", False),
    (7, 3080, 50, F32, False, None, "silu", False),
    (8, 1536, 41, BF16, False, False, "gelu", True),
    (3, 1024, 9, BF16, False, None, "gelu", False),          # few rows, slopes kept
    (4400, 520, 2100, BF16, False, False, "gelu", True),     # tiles of two CTAs, the last one's second without rows
    (2050, 4100, 1000, F16, False, None, None, False),
    (4500, 600, 2056, BF16, True, True, "silu", False),
    (130, 64, 40, BF16, True, True, "gelu", True),           # z kept, for the bias's gradient in float32
]


@pytest.mark.parametrize("M,K,N,dtype,wide,bias,act,residual", CASES)
def test_linear(M, K, N, dtype, wide, bias, act, residual):
    import boost_and_broadside_b200 as bnb
    from boost_and_broadside_b200 import _capi

    g = torch.Generator().manual_seed(M + K)
    x, dy, r = (torch.randn(*s, generator=g).to(dtype) for s in ((M, K), (M, N), (M, N)))
    w = (torch.randn(N, K, generator=g) * K ** -0.5).to(dtype)
    b = None if bias is None else torch.randn(N, generator=g).to(F32 if bias else dtype)
    r = r if residual else None
    want = _bounds(x, w, b, r, dy, act)
    dev = lambda t: None if t is None else t.to(DEV).requires_grad_(True)  # noqa: E731
    xg, wg, bg, rg = dev(x), dev(w.float() if wide else w), dev(b), dev(r)
    leaves = [t for t in (xg, wg, bg, rg) if t is not None]
    call = lambda: bnb.linear(xg, wg, bg, activation=act, residual=rg)  # noqa: E731
    y = call()
    assert y.dtype == dtype
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    assert all(a.dtype == t.dtype for a, t in zip(got, leaves))
    for name, a, (v, e) in zip(("y", "dx", "dw", "db"), (y, *got), want if b is not None else want[:3]):
        _within(a, v, e, name)
    if residual:
        assert torch.equal(got[-1], dy.to(DEV))
    with torch.no_grad():
        assert torch.equal(call(), y)
    again = torch.autograd.grad(call(), leaves, dy.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for i, leaf in enumerate(leaves):                       # one gradient alone is the same
        assert torch.equal(torch.autograd.grad(call(), [leaf], dy.to(DEV))[0], got[i])
    torch.cuda.synchronize()
    assert _capi.lib.bnb_last_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layouts_and_empty_batches(dtype):
    """Leading dims, columns of a wider tensor at an odd offset, transposed weights, an expanded row and gradient, no leading dimension, no rows."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(2)
    K, N = 40, 56
    for act in (None, "gelu"):
        big = torch.randn(3, 5, K + N + 9, generator=g).to(dtype).to(DEV)
        x, r = big[..., 3:3 + K].requires_grad_(True), big[..., 6 + K:6 + K + N].detach().requires_grad_(True)
        w, b = torch.randn(K, N, generator=g).to(DEV).t().requires_grad_(True), torch.randn(2 * N, generator=g).to(DEV)[::2].requires_grad_(True)
        y = bnb.linear(x, w, b, activation=act, residual=r)
        dense = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in (x, w, b, r)]
        z = bnb.linear(*dense[:3], activation=act, residual=dense[3])
        assert y.shape == (3, 5, N) and torch.equal(y, z)
        for dy in (torch.randn(3, 5, N, generator=g).to(dtype).to(DEV), torch.ones((), dtype=dtype, device=DEV).expand(3, 5, N),
                   torch.randn(3, 5, N + 3, generator=g).to(dtype).to(DEV)[..., 1:1 + N]):
            for p, q in zip(torch.autograd.grad(y, [x, w, b, r], dy, retain_graph=True), torch.autograd.grad(z, dense, dy.contiguous(), retain_graph=True)):
                assert torch.equal(p, q)
        row = torch.randn(1, K, generator=g).to(dtype).to(DEV).requires_grad_(True)
        many = row.detach().expand(200, K).contiguous()
        assert torch.equal(bnb.linear(row.expand(200, K), w, b, activation=act), bnb.linear(many, w, b, activation=act))
        flat = bnb.linear(row[0], w, b, activation=act)
        assert flat.shape == (N,) and torch.autograd.grad(flat.sum(), [row])[0].shape == (1, K)
        none = torch.zeros(0, 4, K, dtype=dtype, device=DEV, requires_grad=True)
        y = bnb.linear(none, w, b, activation=act)
        assert y.shape == (0, 4, N)
        grads = torch.autograd.grad(y, [none, w, b], torch.zeros_like(y))
        assert grads[0].shape == none.shape and not any(v.any() for v in grads[1:])


def test_few_rows_of_a_wider_tensor():
    """Rows off every boundary, an expanded one, and weights off theirs, are the same numbers."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(8)
    for dtype in (BF16, F32):
        big = torch.randn(3, 1024 + 11, generator=g).to(dtype).to(DEV)
        w = torch.randn(20 * 1024 + 8, generator=g).to(dtype).to(DEV)
        x, r = big[:, 5:1029], torch.randn(3, 31, generator=g).to(dtype).to(DEV)[:, 7:27]
        y = bnb.linear(x, w[:20480].view(20, 1024), activation="silu", residual=r)
        assert torch.equal(y, bnb.linear(x.contiguous(), w[:20480].view(20, 1024), activation="silu", residual=r.contiguous()))
        off = torch.cat([w[:1], w[:20480]])[1:].view(20, 1024)                # not on 16 bytes: tiles
        assert torch.allclose(bnb.linear(x, off, activation="silu", residual=r).float(), y.float(), rtol=torch.finfo(dtype).eps, atol=1e-3 if dtype == F32 else 1e-2)
        one = bnb.linear(x[:1].expand(3, 1024), w[:20480].view(20, 1024))
        assert torch.equal(one[0], one[1]) and torch.equal(one[0], one[2])
        assert bnb.linear(x[:0], w[:20480].view(20, 1024)).shape == (0, 20)


def test_small_slopes():
    """Slopes from 1 to 4e-11 through what is kept of a bfloat16 call: relative 2^-12, a rounding as the operand dz and one as dx (2^-9 each, and their product), the
    logistic's and its factor's in float32 (s (1 + |z|) 2^-20), and half a step of the smallest numbers kept, 2^-25 2^-15."""
    import boost_and_broadside_b200 as bnb

    x = -torch.linspace(-3, 27, 301).to(BF16)[:, None]
    one = torch.ones(1, 1, dtype=BF16, device=DEV)
    leaf = x.to(DEV).requires_grad_(True)
    got = torch.autograd.grad(bnb.linear(leaf, one, activation="silu"), [leaf], torch.ones(301, 1, dtype=BF16, device=DEV))[0]
    z = x.double()
    s = torch.sigmoid(z)
    d = s * (1 + z * (1 - s))
    _within(got, d, (2 ** -8 + 2 ** -11) * d.abs() + s * (1 + z.abs()) * 2 ** -20 + 2 ** -40, "dx")


def test_gradient_against_differences():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(3)
    for M, K, N, act in ((50, 24, 40, "gelu"), (9, 600, 30, "silu"), (33, 17, 3, None)):
        ins = [torch.randn(*s, generator=g, dtype=torch.float64) * f for s, f in (((M, K), 1), ((N, K), K ** -0.5), ((N,), 1), ((M, N), 1))]
        way = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in ins]
        dy = torch.randn(M, N, generator=g, dtype=torch.float64)
        at = lambda e: float((O.linear(*[t + e * v for t, v in zip(ins[:3], way)], act, ins[3] + e * way[3]) * dy).sum())  # noqa: E731
        slope = (at(1e-5) - at(-1e-5)) / 2e-5
        leaves = [t.float().to(DEV).requires_grad_(True) for t in ins]
        grads = torch.autograd.grad(bnb.linear(*leaves[:3], activation=act, residual=leaves[3]), leaves, dy.float().to(DEV))
        parts = [(a.double().cpu() * v) for a, v in zip(grads, way)]
        assert abs(sum(float(p.sum()) for p in parts) - slope) <= 1e-5 * sum(float(p.abs().sum()) for p in parts)


def test_captured_compiled_and_second_order():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(5)
    for M, K, N in ((70, 64, 96), (6, 2000, 64)):
        x = torch.randn(M, K, generator=g).to(BF16).to(DEV).requires_grad_(True)
        w = (torch.randn(N, K, generator=g) * K ** -0.5).to(DEV).requires_grad_(True)
        b = torch.randn(N, generator=g).to(DEV).requires_grad_(True)
        r, dy = (torch.randn(M, N, generator=g).to(BF16).to(DEV) for _ in range(2))
        r.requires_grad_(True)
        leaves = [x, w, b, r]
        block = lambda x, w, b, r: bnb.linear(x, w, b, activation="silu", residual=r)  # noqa: E731

        def run():
            y = block(*leaves)
            return y.detach(), *torch.autograd.grad(y, leaves, dy)

        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run()
        with torch.no_grad():
            x.copy_(torch.randn(M, K, generator=g))
            w.mul_(1.5)
            b.neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, run()))
        y, z = block(*leaves), torch.compile(block, fullgraph=True)(*leaves)
        assert torch.equal(y, z)
        for a, c in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(z, leaves, dy)):
            assert torch.equal(a, c)
        first, = torch.autograd.grad(block(*leaves), [x], dy, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(first.float().sum(), [w])
    with torch.autograd.graph.save_on_cpu():
        y = block(*leaves)
    for a, c in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(block(*leaves), leaves, dy)):
        assert torch.equal(a, c)


def test_what_is_not_finite_stays_in_its_rows():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(6)
    for dtype in (BF16, F32):
        x, w, dy = (torch.randn(*s, generator=g).to(dtype).to(DEV) for s in ((300, 64), (100, 64), (300, 100)))
        for act in (None, "gelu", "silu"):
            bad = x.clone()
            bad[7, 3] = float("nan")
            bad.requires_grad_(True)
            y = bnb.linear(bad, w, activation=act)
            assert y[7].isnan().all() and y.isfinite().all(1).sum() == 299
            spoiled = dy.clone()
            spoiled[9, 0] = float("inf")
            grad, = torch.autograd.grad(y, [bad], spoiled)
            assert not grad[9].isfinite().any() and grad[10:].isfinite().all() and grad[:7].isfinite().all()


def test_large_products_in_a_graph():
    """Tiles of two CTAs, several launches behind one another, captured and replayed with other numbers, beside the same call on another stream."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(21)
    M, K, N = 4400, 640, 2100
    x, w, b, dy = [torch.randn(*s, generator=g).to(BF16).to(DEV) for s in ((M, K), (N, K), (N,), (M, N))]
    leaves = [t.requires_grad_(True) for t in (x, w, b)]

    def call():
        y = bnb.linear(*leaves, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for scale in (1.0, -0.5):
        with torch.no_grad():
            x.mul_(scale)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            other = call()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, other)) and all(torch.equal(a, e) for a, e in zip(got, call()))
