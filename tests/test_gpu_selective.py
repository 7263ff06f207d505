"""The recurrent operators outside the trunk against their 64-bit implementations: values, states and gradients at the sizes, types,
strides and masks where kernels go wrong, the single-token forms against the sequence forms, and calls under graphs, streams and
compilers.

Tolerances.  A result in a 16-bit type is off by half a step of its type relative to its value, and by what float32 arithmetic
adds, counted relative to the sizes of the terms it is made of: the same formulas with every term's absolute value
(``_conv_sizes``, ``_scan_sizes``).  An operation of a step errs by about 2^-23 and a step has four in a row, so a step by 2^-21
of its size and T steps by T 2^-21; in 16-bit calls the step size p is good to 4e-6, below 2^-17, and so is all that follows from it.  An error
of p or a moves the exponential by its argument's size times as much.  A sum over n terms adds n 2^-24.
"""

import pytest
import torch

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, want, size, steps, terms=1, what=""):
    """size: of the terms, elementwise; steps: in a row; terms: of a sum."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.numel() == 0:
        return
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    unit = 2.0 ** -21 if got.dtype == torch.float32 and not CALL_IS_16[0] else 2.0 ** -17
    want = want.detach()
    err = (got.detach().cpu().double() - want).abs()
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37   # half a step of the subnormal numbers; those of float32 are flushed
    bound = half * want.abs() + tiny + (unit * (steps + 4) + terms * 2.0 ** -24) * size.detach()
    assert bool((err <= bound).all()), f"{what}: off by {float(err[err > bound].max()):.3g} where {float(bound[err > bound].min()):.3g} is allowed"


CALL_IS_16 = [False]   # the call under test has 16-bit activations: its float32 results carry their step size


def _conv_sizes(x, w, b, state, done, lengths, dy, ds):
    """Sizes of y, state, dx, dw, db, dstate."""
    ab = [None if t is None else t.double().abs() for t in (x, w, b, state)]
    leaves = [None if t is None else t.requires_grad_(True) for t in ab]
    pre, st = O.causal_conv(*leaves, done, lengths)
    given = [t for t in leaves if t is not None]
    # |silu'| <= 1.1 and |silu''| <= 0.5
    grads = iter(_oracle_grads([pre, st], given, [dy.double().abs() * (1.1 + pre.detach()), ds.abs()]))
    return [1.1 * pre, st, *(None if t is None else next(grads) for t in leaves)]


def _scan_sizes(u, delta, A, B, C, D, z, bias, state, softplus, done, lengths, dy, ds):
    """Sizes of y, state and the gradients of u, delta, A, B, C, D, z, delta_bias, state."""
    ab = lambda t: 0.0 if t is None else t.double().abs()  # noqa: E731
    T, R, W = u.shape
    G, N = B.shape[-2:]
    share = lambda t: ab(t).repeat_interleave(W // G, 1)  # noqa: E731
    group = lambda t: t.unflatten(1, (G, W // G)).sum(2)  # noqa: E731
    raw = delta.double() + (0.0 if bias is None else bias.double())
    p = torch.nn.functional.softplus(raw, threshold=50.0) if softplus else raw
    sp = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    arg = p[..., None] * A.double()
    e = torch.exp(arg) * (1 + arg.abs())
    p = p.abs()
    sg = torch.ones_like(p) if z is None else torch.sigmoid(z.double())
    gate = torch.ones_like(p) if z is None else ab(z) * sg
    slope = torch.zeros_like(p) if z is None else sg * (1 + ab(z) * (1 - sg))
    live = torch.ones(T, R, dtype=torch.bool) if lengths is None else torch.arange(T)[:, None] < lengths[None]
    h = torch.zeros(R, W, N, dtype=torch.float64) + ab(state)
    before, ys, y = [], [], torch.zeros(T, R, W, dtype=torch.float64)
    for t in range(T):
        start = h if t == 0 or done is None else torch.where(done[t - 1][:, None, None], 0.0, h)
        before.append(start)
        new = e[t] * start + (p[t] * ab(u[t]))[..., None] * share(B[t])
        ys.append((new * share(C[t])).sum(-1) + ab(D) * ab(u[t]))
        y[t] = torch.where(live[t][:, None], ys[t] * gate[t], 0.0)
        h = torch.where(live[t][:, None, None], new, h)
    out = h
    du, dd, dz, db, dc = (torch.zeros(t.shape, dtype=torch.float64) for t in (u, delta, u, B, C))
    dA, dD, dbias = torch.zeros(W, N, dtype=torch.float64), torch.zeros(W, dtype=torch.float64), torch.zeros(W, dtype=torch.float64)
    carry = ab(ds)
    for t in range(T - 1, -1, -1):
        on = live[t][:, None]
        dyv = torch.where(on, ab(dy[t]) * gate[t], 0.0)
        Bt, Ct, pu = share(B[t]), share(C[t]), p[t] * ab(u[t])
        new = e[t] * before[t] + pu[..., None] * Bt
        gh = carry + Ct * dyv[..., None]
        ghe = gh * e[t] * before[t]
        ghb = (gh * Bt).sum(-1)
        draw = torch.where(on, ((ghe * ab(A)).sum(-1) + ghb * ab(u[t])) * sp[t], 0.0)
        du[t] = torch.where(on, ghb * p[t] + ab(D) * dyv, 0.0)
        dd[t] = draw
        dz[t] = torch.where(on, ab(dy[t]) * ys[t] * slope[t], 0.0)
        dc[t] = group(dyv[..., None] * new)
        db[t] = group(torch.where(on[..., None], gh * pu[..., None], 0.0))
        dA += torch.where(on[..., None], ghe * p[t][..., None], 0.0).sum(0)
        dD += (dyv * ab(u[t])).sum(0)
        dbias += draw.sum(0)
        back = gh * e[t]
        if t > 0 and done is not None:
            back = torch.where(done[t - 1][:, None, None], 0.0, back)
        carry = torch.where(on[..., None], back, carry)
    return [y, out, du, dd, dA, db, dc, dD, dz, dbias, carry]


def _r(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def _layout(t, how):
    """The same values on the device: dense, as columns of a wider tensor, batch-major, or at an odd offset."""
    if how == "dense":
        return t.to(DEV)
    if how == "columns":
        wide = torch.full((*t.shape[:-1], t.shape[-1] + 5), float("nan"), dtype=t.dtype)
        wide[..., 3:3 + t.shape[-1]] = t
        return wide.to(DEV)[..., 3:3 + t.shape[-1]]
    return t.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)


def _masks(g, T, R, masks):
    done = torch.rand(T, R, generator=g) < 0.2 if "done" in masks else None
    lengths = None
    if "ragged" in masks:
        lengths = torch.randint(0, T + 1, (R,), generator=g)
        lengths[0] = T
        if R > 1:
            lengths[1] = 0
        if R > 2:
            lengths[2] = 1
    return done, lengths


def _nan_behind(t, lengths):
    """What stands behind a row's end is never looked at."""
    if lengths is None:
        return t
    t = t.clone()
    for r, n in enumerate(lengths.tolist()):
        t[n:, r] = float("nan")
    return t


def _oracle_grads(outs, leaves, given):
    """Zeros for what an output does not depend on (sequences without steps)."""
    pairs = [(o, g.double()) for o, g in zip(outs, given) if o.requires_grad]
    got = torch.autograd.grad([o for o, _ in pairs], leaves, [g for _, g in pairs], allow_unused=True)
    return [torch.zeros_like(v) if w is None else w for w, v in zip(got, leaves)]


def _dev(*ts):
    return [None if t is None else t.to(DEV) for t in ts]


# ----------------------------------------------------------------------------- causal convolution


CONV = [
    # T, R, C, K, type, layout, masks, activation
    (1, 1, 1, 2, torch.float32, "dense", "", None),
    (0, 3, 8, 4, torch.bfloat16, "dense", "", "silu"),
    (2, 3, 8, 4, torch.float32, "dense", "done", "silu"),
    (3, 5, 64, 4, torch.bfloat16, "dense", "ragged", "silu"),
    (16, 7, 24, 3, torch.float16, "batch", "done ragged", "silu"),
    (17, 4, 33, 4, torch.bfloat16, "columns", "done ragged", "silu"),
    (33, 2, 520, 2, torch.float32, "batch", "done", None),
    (100, 3, 72, 4, torch.bfloat16, "dense", "done ragged", "silu"),
    (67, 9, 31, 4, torch.float32, "columns", "ragged", "silu"),
    (5, 300, 40, 4, torch.float16, "dense", "done", None),
]


@pytest.mark.parametrize("T,R,C,K,dtype,layout,masks,act", CONV)
@pytest.mark.parametrize("with_state", [True, False])
def test_causal_conv(T, R, C, K, dtype, layout, masks, act, with_state):
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(T + R)
    x, w, b = _r(g, T, R, C, dtype=dtype), _r(g, C, K), _r(g, C) if with_state else None
    state = _r(g, R, K - 1, C) if with_state else None
    done, lengths = _masks(g, T, R, masks)
    dy, ds = _r(g, T, R, C, dtype=dtype), _r(g, R, K - 1, C)
    leaves = [t for t in (x, w, b, state) if t is not None]
    want_leaves = [t.double().requires_grad_(True) for t in leaves]
    it = iter(want_leaves)
    wy, wst = O.causal_conv(next(it), next(it), next(it) if b is not None else None, next(it) if state is not None else None, done, lengths, act)
    want = _oracle_grads([wy, wst], want_leaves, [dy, ds])

    xd = _layout(_nan_behind(x, lengths), layout).requires_grad_(True)
    wd, bd, sd = [None if t is None else t.to(DEV).requires_grad_(True) for t in (w, b, state)]
    y, st = bnb.causal_conv(xd, wd, bd, state=sd, done=_dev(done)[0], lengths=_dev(lengths)[0], activation=act)
    got = torch.autograd.grad([y, st], [t for t in (xd, wd, bd, sd) if t is not None], [_layout(_nan_behind(dy, lengths), layout), ds.to(DEV)])
    assert y.dtype == dtype and st.dtype == torch.float32
    CALL_IS_16[0] = False   # no step sizes here
    sy, sst, *sizes = _conv_sizes(x, w, b, state, done, lengths, dy, ds)
    _close(y, wy, sy, 1, what="y")
    assert torch.equal(st.cpu().double(), wst.detach())   # copies
    names, sums = ["x", "weight", "bias", "state"], [1, T * R, T * R, 1]
    for name, a, v, sz, n in zip([m for m, t in zip(names, (x, w, b, state)) if t is not None], got, want, [t for t in sizes if t is not None],
                                 [n for n, t in zip(sums, (x, w, b, state)) if t is not None]):
        _close(a, v, sz, 2, n, what="d " + name)
    with torch.no_grad():
        y2, _ = bnb.causal_conv(xd, wd, bd, state=sd, done=_dev(done)[0], lengths=_dev(lengths)[0], activation=act)
    assert torch.equal(y2, y)


@pytest.mark.parametrize("K,dtype", [(4, torch.bfloat16), (2, torch.float32), (3, torch.float16)])
def test_conv_steps_are_the_sequence(K, dtype):
    """Single tokens with the state in place, episodes cleared by `reset`, give the sequence's values."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(K)
    T, R, C = 6, 11, 40
    x, w, b, state = _r(g, T, R, C, dtype=dtype).to(DEV), _r(g, C, K).to(DEV), _r(g, C).to(DEV), _r(g, R, K - 1, C).to(DEV)
    done = (torch.rand(T, R, generator=g) < 0.3).to(DEV)
    y, st = bnb.causal_conv(x, w, b, state=state, done=done, activation="silu")
    held = state.clone()
    for t in range(T):
        got = bnb.causal_conv_step(x[t], held, w, b, reset=done[t - 1] if t else None, activation="silu")
        assert torch.equal(got, y[t])
    assert torch.equal(held, st)


# ----------------------------------------------------------------------------- selective scan


SCAN = [
    # T, R, W, N, G, type, layout, masks
    (1, 1, 1, 1, 1, torch.float32, "dense", ""),
    (0, 2, 8, 16, 1, torch.bfloat16, "dense", ""),
    (2, 3, 32, 4, 1, torch.float32, "dense", "done"),
    (7, 4, 33, 16, 1, torch.bfloat16, "columns", "done ragged"),
    (8, 3, 64, 16, 1, torch.float32, "dense", "done ragged"),
    (9, 5, 40, 8, 2, torch.float16, "batch", "ragged"),
    (17, 2, 130, 16, 2, torch.float32, "batch", "done ragged"),
    (33, 3, 66, 11, 2, torch.bfloat16, "columns", "done"),
    (40, 2, 24, 32, 1, torch.float32, "dense", "done"),
    (25, 3, 20, 64, 4, torch.float16, "dense", "ragged"),
    (31, 2, 9, 2, 3, torch.float32, "columns", "done ragged"),
    (16, 70, 72, 16, 1, torch.bfloat16, "dense", "done ragged"),
    (200, 2, 40, 16, 1, torch.float32, "batch", "done ragged"),      # several splits of time
    (333, 1, 70, 5, 1, torch.bfloat16, "dense", ""),
    (261, 3, 12, 64, 1, torch.float32, "dense", "done ragged"),
    (20, 700, 8, 16, 1, torch.bfloat16, "dense", "done ragged"),     # more rows than are worked on at once, some without steps
    (11, 650, 3, 3, 1, torch.float32, "columns", "ragged"),
    (9, 610, 16, 64, 1, torch.float16, "batch", "done ragged"),
]


def _scan_inputs(g, T, R, W, N, G, dtype):
    u, delta, z = (_r(g, T, R, W, dtype=dtype) for _ in range(3))
    B, C = (_r(g, T, R, G, N, dtype=dtype) for _ in range(2))
    A = -torch.rand(W, N, generator=g) * 4 - 0.05
    return u, delta, A, B, C, _r(g, W), z, _r(g, W) - 1.0, _r(g, R, W, N)


def _flat_layout(t, how):
    """B and C: the layouts above over their last two dims as columns."""
    return _layout(t.flatten(-2), how).unflatten(-1, t.shape[-2:])


@pytest.mark.parametrize("T,R,W,N,G,dtype,layout,masks", SCAN)
@pytest.mark.parametrize("full", [True, False])
def test_selective_scan(T, R, W, N, G, dtype, layout, masks, full):
    """full: with skip, gate, bias, softplus and a given state; otherwise none of them."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(7 * T + R)
    inputs = list(_scan_inputs(g, T, R, W, N, G, dtype))
    if not full:
        inputs[1] = (0.2 * torch.rand(T, R, W, generator=g)).to(dtype)
        inputs[5] = inputs[6] = inputs[7] = inputs[8] = None
    done, lengths = _masks(g, T, R, masks)
    dy, ds = _r(g, T, R, W, dtype=dtype), _r(g, R, W, N)
    wl = [None if t is None else t.double().requires_grad_(True) for t in inputs]
    wy, wst = O.selective_scan(*wl[:8], softplus=full, state=wl[8], done=done, lengths=lengths)
    given = [t for t in wl if t is not None]
    want = _oracle_grads([wy, wst], given, [dy, ds])

    leaves = []
    for i, t in enumerate(inputs):
        if t is None:
            leaves.append(None)
        elif i in (0, 1, 6):
            leaves.append(_layout(_nan_behind(t, lengths), layout).requires_grad_(True))
        elif i in (3, 4):
            leaves.append(_flat_layout(_nan_behind(t, lengths), layout).requires_grad_(True))
        else:
            leaves.append(t.to(DEV).requires_grad_(True))
    u, delta, A, B, C, D, z, bias, state = leaves
    kwargs = dict(z=z, delta_bias=bias, softplus=full, state=state, done=_dev(done)[0], lengths=_dev(lengths)[0])
    y, st = bnb.selective_scan(u, delta, A, B, C, D, **kwargs)
    got = torch.autograd.grad([y, st], [t for t in leaves if t is not None], [_layout(_nan_behind(dy, lengths), layout), ds.to(DEV)])
    CALL_IS_16[0] = dtype != torch.float32
    sy, sst, *sizes = _scan_sizes(*inputs, full, done, lengths, dy, ds)
    _close(y, wy, sy, T, N, what="y")
    _close(st, wst, sst, T, what="state")
    names = ["u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"]
    terms = [N, N, T * R, W, W, T * R, N, T * R * N, 1]
    for (name, n, sz), a, v in zip([(m, k, q) for m, k, q, t in zip(names, terms, sizes, leaves) if t is not None], got, want):
        _close(a, v, sz, 2 * T, n, what="d " + name)
    with torch.no_grad():
        y2, st2 = bnb.selective_scan(u, delta, A, B, C, D, **kwargs)
    assert torch.equal(y2, y) and torch.equal(st2, st)
    again = torch.autograd.grad(bnb.selective_scan(u, delta, A, B, C, D, **kwargs), [t for t in leaves if t is not None],
                                [_layout(_nan_behind(dy, lengths), layout), ds.to(DEV)])
    assert all(torch.equal(a, b) for a, b in zip(again, got))   # sums in a fixed order


@pytest.mark.parametrize("first,behind", [(8, 16), (6, 18)])
def test_an_ended_episode_keeps_its_values(first, behind):
    """Infinities and NaN of an episode, its gradients' too, do not reach the next or the last one's values.  The gradients of B and C
    are the exception that is documented: they may within eight steps."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(21)
    T, R, W, N = 24, 3, 40, 16
    u, delta, A, B, C, D, z, bias, state = [t.to(DEV) for t in _scan_inputs(g, T, R, W, N, 1, torch.float32)]
    done = torch.zeros(T, R, dtype=torch.bool, device=DEV)
    done[first - 1] = done[behind - 1] = True
    dy = _r(g, T, R, W).to(DEV)
    runs = []
    for value in (0.0, float("nan"), float("inf")):
        v, gy = u.clone(), dy.clone()
        v[10, :, 3] = value
        gy[12, :, 5] = value
        leaves = [t.clone().requires_grad_(True) for t in (v, delta, z, B, C, state)]
        y, st = bnb.selective_scan(leaves[0], leaves[1], A, leaves[3], leaves[4], D, z=leaves[2], delta_bias=bias, softplus=True, state=leaves[5], done=done)
        runs.append([y, *torch.autograd.grad([y, st], leaves, [gy, torch.ones_like(st)]), st])
    for other in runs[1:]:
        for a, b in zip(runs[0][:4], other[:4]):   # per step: y and the gradients of u, delta, z
            assert torch.equal(a[:first], b[:first]) and torch.equal(a[behind:], b[behind:])
        for a, b in zip(runs[0][4:6], other[4:6]):
            lo, hi = first // 8 * 8, (behind + 7) // 8 * 8
            assert torch.equal(a[:lo], b[:lo]) and torch.equal(a[hi:], b[hi:])
        assert torch.equal(runs[0][6], other[6]) and torch.equal(runs[0][7], other[7])


def test_the_same_tensor_twice():
    """u as step sizes too, B as C too: the gradients add up."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(22)
    T, R, W, N = 13, 4, 24, 8
    u, _, A, B, *_ = _scan_inputs(g, T, R, W, N, 1, torch.float32)
    dy = _r(g, T, R, W)
    ud, Bd = u.to(DEV).requires_grad_(True), B.to(DEV).requires_grad_(True)
    got = torch.autograd.grad(bnb.selective_scan(ud, ud, A.to(DEV), Bd, Bd, softplus=True)[0], [ud, Bd], dy.to(DEV))
    one, two, b, c = [t.to(DEV).requires_grad_(True) for t in (u, u, B, B)]
    apart = torch.autograd.grad(bnb.selective_scan(one, two, A.to(DEV), b, c, softplus=True)[0], [one, two, b, c], dy.to(DEV))
    assert torch.equal(got[0], apart[0] + apart[1]) and torch.equal(got[1], apart[2] + apart[3])


def test_scan_gradient_against_differences():
    """The derivative along a random direction in float32 against a central difference of the 64-bit forward."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(3)
    T, R, W, N, G = 12, 3, 10, 6, 2
    inputs = [t.double() for t in _scan_inputs(g, T, R, W, N, G, torch.float32)]
    done = torch.rand(T, R, generator=g) < 0.2
    dy, ds = _r(g, T, R, W), _r(g, R, W, N)
    way = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in inputs]

    def loss(at):
        y, st = O.selective_scan(*at[:8], softplus=True, state=at[8], done=done)
        return float((y * dy).sum() + (st * ds).sum())

    eps = 1e-5
    slope = (loss([t + eps * v for t, v in zip(inputs, way)]) - loss([t - eps * v for t, v in zip(inputs, way)])) / (2 * eps)
    leaves = [t.float().to(DEV).requires_grad_(True) for t in inputs]
    u, delta, A, B, C, D, z, bias, state = leaves
    outs = bnb.selective_scan(u, delta, A, B, C, D, z=z, delta_bias=bias, softplus=True, state=state, done=done.to(DEV))
    grads = torch.autograd.grad(outs, leaves, [dy.to(DEV), ds.to(DEV)])
    got = sum(float((a.double().cpu() * v).sum()) for a, v in zip(grads, way))
    size = sum(float((a.double().cpu() * v).abs().sum()) for a, v in zip(grads, way))
    assert abs(got - slope) <= 1e-5 * size   # 16 steps of 2^-21 relative to the terms; the difference itself is good to 1e-8


@pytest.mark.parametrize("N,G,dtype", [(16, 1, torch.bfloat16), (6, 2, torch.float32), (64, 1, torch.float16), (1, 1, torch.float32), (32, 3, torch.bfloat16)])
@pytest.mark.parametrize("R", [1, 5, 2500])
def test_scan_steps_are_the_sequence(N, G, dtype, R):
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(N)
    T, W = 3, 36
    u, delta, A, B, C, D, z, bias, state = _scan_inputs(g, T, R, W, N, G, dtype)
    done = torch.rand(T, R, generator=g) < 0.3
    wy, wst = O.selective_scan(u, delta, A, B, C, D, z, bias, True, state, done)
    held = state.to(DEV)
    args = _dev(A, D, bias)
    CALL_IS_16[0] = dtype != torch.float32
    sy, sst, *_ = _scan_sizes(u, delta, A, B, C, D, z, bias, state, True, done, None, torch.zeros(T, R, W), torch.zeros(R, W, N))
    for t in range(T):
        ut, zt = torch.cat([u[t], z[t]], -1).to(DEV).split(W, -1)
        got = bnb.selective_step(ut, delta[t].to(DEV), args[0], B[t].to(DEV), C[t].to(DEV), args[1], held, z=zt, delta_bias=args[2], softplus=True,
                                 reset=done[t - 1].to(DEV) if t else None)
        _close(got, wy[t], sy[t], T, N, what=f"y {t}")
    _close(held, wst, sst, T, what="state")


def test_large_and_extreme_steps():
    """Steps so large that the decay underflows to 0, zero steps, growing states and values next to softplus' threshold."""
    import boost_and_broadside_b200 as bnb

    T, R, W, N = 5, 2, 8, 4
    g = torch.Generator().manual_seed(1)
    u, delta, A, B, C, D, z, bias, state = _scan_inputs(g, T, R, W, N, 1, torch.float32)
    delta = torch.tensor([-200.0, -30.0, -3.0, 0.0, 19.5, 20.5, 300.0, 3000.0]).expand(T, R, W).contiguous()
    A[:, 0] = 0.0
    wy, wst = O.selective_scan(u, delta, A, B, C, D, z, None, True, state)
    y, st = bnb.selective_scan(*_dev(u, delta, A, B, C, D), z=z.to(DEV), softplus=True, state=state.to(DEV))
    CALL_IS_16[0] = False
    sy, sst, *_ = _scan_sizes(u, delta, A, B, C, D, z, None, state, True, None, None, torch.zeros(T, R, W), torch.zeros(R, W, N))
    _close(y, wy, sy, T, N, what="y")
    _close(st, wst, sst, T, what="state")


def test_captured_calls_replay_and_do_not_share():
    """Two captured graphs of forward and backward on two streams, replayed in turn with new inputs, give the eager results."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(5)
    graphs = []
    for k, (T, R, W, N) in enumerate([(300, 2, 40, 16), (24, 6, 96, 8)]):
        stream = torch.cuda.Stream()
        ins = [t.to(DEV) for t in _scan_inputs(g, T, R, W, N, 1, torch.float32)]
        w = _r(g, W, 4).to(DEV).requires_grad_(True)

        def run(ins=ins, w=w):
            x, _ = bnb.causal_conv(ins[0], w, activation="silu")
            y, st = bnb.selective_scan(x, *ins[1:6], z=ins[6], delta_bias=ins[7], softplus=True, state=ins[8])
            return y.detach(), st.detach(), *torch.autograd.grad([y, st], [w, ins[2]], [ins[1], ins[8]])

        ins[2].requires_grad_(True)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run()
        graphs.append((graph, ins, run, out))
    for round_ in range(2):
        for _, ins, _, _ in graphs:
            ins[0].copy_(_r(g, *ins[0].shape))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, _, run, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, run()))


def test_under_torch_compile_and_second_order():
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(6)
    T, R, W, N = 20, 3, 24, 8
    ins = [t.to(DEV) for t in _scan_inputs(g, T, R, W, N, 1, torch.bfloat16)]
    w = _r(g, W, 4).to(DEV)
    for t in (*ins, w):
        t.requires_grad_(True)
    dy = _r(g, T, R, W, dtype=torch.bfloat16).to(DEV)

    def layer(x, w):
        x, taps = bnb.causal_conv(x, w, activation="silu")
        y, st = bnb.selective_scan(x, *ins[1:6], z=ins[6], delta_bias=ins[7], softplus=True, state=ins[8])
        return y, st, taps

    eager = layer(ins[0], w)
    compiled = torch.compile(layer, fullgraph=True)(ins[0], w)
    assert all(torch.equal(a, b) for a, b in zip(eager, compiled))
    a = torch.autograd.grad(eager[0], [ins[0], w, ins[2], ins[3]], dy)
    b = torch.autograd.grad(compiled[0], [ins[0], w, ins[2], ins[3]], dy)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    y, *_ = layer(ins[0], w)
    first = torch.autograd.grad(y, [w], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        torch.autograd.grad(first[0].sum(), [w])

    taps, held = torch.zeros(R, 3, W, device=DEV), torch.zeros(R, W, N, device=DEV)
    steps = [t.detach() for t in ins]

    def one(x, taps, held):
        x = bnb.causal_conv_step(x, taps, w, activation="silu")
        return bnb.selective_step(x, steps[1][0], steps[2], steps[3][0], steps[4][0], steps[5], held, z=steps[6][0], delta_bias=steps[7], softplus=True)

    with torch.no_grad():
        t1, h1, t2, h2 = taps.clone(), held.clone(), taps.clone(), held.clone()
        want = one(steps[0][0], t1, h1)
        got = torch.compile(one, fullgraph=True)(steps[0][0], t2, h2)
    assert torch.equal(want, got) and torch.equal(t1, t2) and torch.equal(h1, h2)


def test_on_another_stream():
    """The kernels run on the current stream, behind what it holds."""
    import boost_and_broadside_b200 as bnb

    g = torch.Generator().manual_seed(8)
    ins = [t.to(DEV) for t in _scan_inputs(g, 64, 4, 64, 16, 1, torch.float32)]
    want, _ = bnb.selective_scan(*ins[:6], z=ins[6])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(ins[0])
        torch.cuda._sleep(20_000_000)
        late.copy_(ins[0])
        got, _ = bnb.selective_scan(late, *ins[1:6], z=ins[6])
    side.synchronize()
    assert torch.equal(got.view(torch.int32), want.view(torch.int32))   # bits: without softplus the states grow beyond all numbers
