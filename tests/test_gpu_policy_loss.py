"""``policy_loss`` against its 64-bit implementation: slices of one action to tens of thousands, every type, masks, forbidden actions, layouts, its
gradient, captured and compiled calls.

Tolerances are first-order bounds of a float32 evaluation (``oracle.update_oracle.policy_bounds``), elementwise, with half a step of a result's own
type on top; no ratio of the inputs stands within 1e-3 of a border of the clipping, where a rounding would decide the branch."""

import math

import pytest
import torch

from oracle import update_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(R, sizes, dtype, seed=0, forbidden=False, clip=(0.2, 0.2), spread=2.0):
    """logits (R, V), actions (R, S), old, adv, ref: the ratios and the reference follow from the logits."""
    g = torch.Generator().manual_seed(seed + R)
    V = sum(sizes)
    z = (spread * torch.randn(R, V, generator=g)).to(dtype)
    acts = torch.stack([torch.randint(n, (R,), generator=g) for n in sizes], 1)
    first = torch.tensor([sum(sizes[:i]) for i in range(len(sizes))])
    if forbidden:
        off = (torch.rand(R, V, generator=g) < 0.3).scatter_(1, acts + first, False)
        low = torch.where(torch.rand(R, V, generator=g) < 0.5, -math.inf, torch.finfo(dtype).min).to(dtype)
        z = torch.where(off, low, z)
    _, l, _ = O.policy_loss(z, acts, torch.zeros(R), torch.zeros(R), sizes=sizes)
    moved = 0.25 * torch.randn(R, generator=g, dtype=torch.float64)
    for border in (1 - clip[0], 1 + clip[1]):
        moved = torch.where((moved.exp() - border).abs() < 1e-3, moved + 0.01, moved)
    ref = (l + 0.3 * torch.randn(R, generator=g, dtype=torch.float64)).float()
    return z, acts, (l - moved).float(), torch.randn(R, generator=g), ref


def _within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if want.numel() == 0:
        return
    err = (got.detach().cpu().double() - want).abs()
    own = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 1e-37
    allowed = 1.1 * (bound + own * want.abs()) + tiny
    assert bool((err <= allowed).all()), f"{what}: off by {float((err / allowed).max()):.2f} times what is allowed"


def _compare(z, acts, old, adv, dtype, weights=None, ref=None, sizes=None, clip=(0.2, 0.2), kl=0.0, ent=0.0, scale=1.0, additions=80):
    import boost_and_broadside_b200 as bnb

    zl = z.double().requires_grad_(True)
    loss, l, stats = O.policy_loss(zl, acts, old, adv, weights, ref, sizes, clip, kl, ent)
    dz, = torch.autograd.grad(loss, [zl], torch.tensor(scale, dtype=torch.float64))
    bounds = O.policy_bounds(z, acts, old, adv, weights, ref, sizes, clip, kl, ent, scale, additions)
    x = z.to(DEV).requires_grad_(True)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    a = acts if sizes is not None else acts[:, 0]
    out = bnb.policy_loss(x, dev(a), dev(old), dev(adv), weights=dev(weights), ref_logprob=dev(ref), sizes=sizes, clip=clip, kl_coef=kl, entropy_coef=ent)
    grad, = torch.autograd.grad(out[0], [x], torch.tensor(scale, device=DEV))
    assert grad.dtype == dtype and [t.requires_grad for t in out] == [True, False, False]
    for name, got, want, bound in zip(("loss", "logprob", "stats", "dlogits"), (*out, grad), (loss.detach(), l.detach(), stats.detach(), dz), bounds):
        _within(got, want, bound, name)
    return out, grad


F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CASES = [
    # rows, sizes (None: one slice), type, weights, reference policy, forbidden actions, loss scale
    (1, [2], F32, None, False, False, 1.0),
    (3, [1], BF16, None, True, False, 1.0),
    (16, [3, 7, 2], F32, "mask", False, False, 1.0),
    (1000, [3, 7, 2], BF16, "mask", True, True, 0.25),
    (129, [3, 7, 2], F16, "float", True, True, 300.0),
    (130, [40, 30, 10, 7], F32, None, False, False, 1.0),            # tiles that take nearly 48 KB of shared memory: with four slices,
    (70, [30, 25, 20, 25, 20, 25, 20, 10], BF16, "mask", True, False, 1.0),   # eight
    (40, [22] * 15 + [19], F16, None, False, True, 80.0),            # and sixteen
    (200, [64], BF16, "float", True, False, 1.0),
    (77, [64, 1, 64, 63, 2, 5, 11, 64, 3], F32, None, True, True, 1.0),
    (50, [5] * 16, F16, "mask", False, False, 100.0),
    (40, [65], F32, "mask", True, False, 3.0),
    (33, [1000], BF16, "mask", True, True, 1.0),
    (21, [70, 3, 201], F16, None, True, True, 64.0),
    (2, [1023], F32, None, False, True, 1.0),
    (9, [1025], BF16, "float", True, False, 1.0),
    (5, [300, 2, 900], F32, "mask", True, True, 1.0),
    (4, [5001], F32, None, True, True, 1.0),
    (3, [40003], BF16, "mask", True, False, 1.0),
    (2, [33001], F16, None, False, True, 8.0),
    (3, [33003], F32, "mask", True, False, 1.0),             # rows of more than 128 KB
    (70, [100], BF16, "float", False, True, 2.0),            # several rows a warp, some of them without weight
    (45, [999], F32, "mask", True, False, 1.0),
]


@pytest.mark.parametrize("R,sizes,dtype,kind,ref,forbidden,scale", CASES)
def test_policy_loss(R, sizes, dtype, kind, ref, forbidden, scale):
    clip = (0.2, 0.3)
    z, acts, old, adv, r = _inputs(R, sizes, dtype, forbidden=forbidden, clip=clip)
    g = torch.Generator().manual_seed(R)
    weights = None
    if kind is not None:
        weights = torch.rand(R, generator=g) < 0.7
        weights[0] = True
        if kind == "float":
            weights = weights * (0.2 + torch.rand(R, generator=g))
        z[~weights.bool()] = math.nan           # rows without weight are not looked at
        acts[~weights.bool()] = -100
    many = sizes if len(sizes) > 1 else None
    longest = max(sizes)
    additions = 40 + (longest if longest <= 64 else longest // 32 if sum(sizes) <= 1024 else longest // 256)
    args = dict(weights=weights, ref=r if ref else None, sizes=many, clip=clip, kl=0.1 if ref else 0.0, ent=0.02, scale=scale, additions=additions)
    _compare(z, acts, old, adv, dtype, **args)
    again = _compare(z, acts, old, adv, dtype, **args)
    for a, b in zip((*again[0], again[1]), (*_compare(z, acts, old, adv, dtype, **args)[0], again[1])):
        assert torch.equal(a, b)


def test_layouts():
    """Leading dimensions, columns of a wider tensor at an odd offset, an expanded row, int32 actions, a plain number as the clipping."""
    import boost_and_broadside_b200 as bnb

    for sizes in ([3, 7, 2], [90], [1111]):
        V, S = sum(sizes), len(sizes)
        z, acts, old, adv, ref = _inputs(10, sizes, BF16)
        wide = torch.full((2, 5, V + 13), math.nan, dtype=BF16, device=DEV)
        wide[..., 5:5 + V] = z.view(2, 5, V).to(DEV)
        x, dense = wide[..., 5:5 + V].requires_grad_(True), z.to(DEV).requires_grad_(True)
        a = acts.view(2, 5, S) if S > 1 else acts.view(2, 5)
        dev = [t.view(2, 5).to(DEV) for t in (old, adv, ref)]
        kw = dict(sizes=sizes if S > 1 else None, clip=0.2, kl_coef=0.1, entropy_coef=0.01)
        # rows that start elsewhere in their 16 bytes are summed in other parts: both results are within the bounds of the exact ones
        bounds = O.policy_bounds(z, acts, old, adv, None, ref, sizes, (0.2, 0.2), 0.1, 0.01, additions=40 + max(sizes) // 16)

        def near(got, want, bound):
            own = torch.finfo(got.dtype).eps / 2
            assert bool(((got.double() - want.double()).abs().cpu() <= 2.2 * (bound + own * want.double().abs().cpu())).all())

        one = bnb.policy_loss(x, a.int().to(DEV), dev[0], dev[1], ref_logprob=dev[2], **kw)
        two = bnb.policy_loss(dense, (acts if S > 1 else acts[:, 0]).to(DEV), *(t.view(-1) for t in dev[:2]), ref_logprob=dev[2].view(-1), **kw)
        assert one[1].shape == (2, 5)
        for p, q, bound in zip(one, two, bounds):
            near(p.detach().reshape(q.shape), q.detach(), bound)
        p, q = torch.autograd.grad(one[0], [x])[0], torch.autograd.grad(two[0], [dense])[0]
        assert p.shape == x.shape
        near(p.reshape(q.shape), q, bounds[3])
        row = z[:1].to(DEV).requires_grad_(True)
        many = z[:1].to(DEV).expand(10, V).contiguous().requires_grad_(True)
        bounds = O.policy_bounds(z[:1].expand(10, V), acts, old, adv, None, None, sizes, (0.2, 0.2), 0.1, 0.01, additions=40 + max(sizes) // 16)
        three, four = (bnb.policy_loss(t, (acts if S > 1 else acts[:, 0]).to(DEV), old.to(DEV), adv.to(DEV), **kw) for t in (row.expand(10, V), many))
        near(three[1], four[1], bounds[1])
        each, = torch.autograd.grad(four[0], [many])
        summed, = torch.autograd.grad(three[0], [row])
        error = bounds[3].sum(0) + torch.finfo(BF16).eps * each.double().abs().sum(0).cpu()     # ten roundings of each side and those of their sums
        assert bool(((summed.double() - each.double().sum(0, keepdim=True)).abs().cpu() <= 6 * error).all())
        flat = z[0].to(DEV).requires_grad_(True)              # no leading dimension: one row
        out = bnb.policy_loss(flat, (acts[0] if S > 1 else acts[0, 0]).to(DEV), old[0].to(DEV), adv[0].to(DEV), **kw)
        assert out[1].shape == () and torch.autograd.grad(out[0], [flat])[0].shape == (V,)


@pytest.mark.parametrize("sizes", [[3, 7, 2], [200], [2500]])
def test_rows_that_nothing_is_left_of(sizes):
    """No rows; no row with weight; an action outside of its slice; a row of forbidden actions only; NaN and infinities in rows of weight."""
    import boost_and_broadside_b200 as bnb

    S, V = len(sizes), sum(sizes)
    kw = dict(sizes=sizes if S > 1 else None, kl_coef=0.1, entropy_coef=0.01)
    z, acts, old, adv, ref = (t.to(DEV) for t in _inputs(6, sizes, F32))
    pick = lambda a: a if S > 1 else a[:, 0]  # noqa: E731
    none = z[:0].clone().requires_grad_(True)
    loss, l, stats = bnb.policy_loss(none, pick(acts)[:0], old[:0], adv[:0], ref_logprob=ref[:0], **kw)
    assert loss.item() == 0 and l.shape == (0,) and not stats.any() and torch.autograd.grad(loss, [none])[0].shape == (0, V)
    x = torch.full_like(z, math.nan).requires_grad_(True)
    loss, l, stats = bnb.policy_loss(x, pick(acts), old, adv, ref_logprob=ref, weights=torch.zeros(6, dtype=torch.bool, device=DEV), **kw)
    assert float(loss) == 0 and not l.any() and not stats.any() and not torch.autograd.grad(loss, [x])[0].any()
    for spoil in ("action", "forbidden", "nan", "inf"):
        bad, a = z.clone(), acts.clone()
        if spoil == "action":
            a[2, -1] = sizes[-1]
            a[4, 0] = -1
        else:
            bad[2], bad[4] = (-math.inf, -math.inf) if spoil == "forbidden" else (z[2], z[4])
            if spoil != "forbidden":
                bad[2, V // 2] = bad[4, V - 1] = math.nan if spoil == "nan" else math.inf
        bad.requires_grad_(True)
        loss, l, _ = bnb.policy_loss(bad, pick(a), old, adv, ref_logprob=ref, **kw)
        grad, = torch.autograd.grad(loss, [bad])
        assert math.isnan(float(loss)) and l.isnan().tolist() == [False, False, True, False, True, False], spoil
        assert grad.isfinite().all(1).tolist() == [True, True, False, True, False, True], spoil
        # the same rows without weight
        w = torch.tensor([1, 1, 0, 1, 0, 1.0], device=DEV)
        loss, l, _ = bnb.policy_loss(bad, pick(a), old, adv, ref_logprob=ref, weights=w, **kw)
        grad, = torch.autograd.grad(loss, [bad])
        assert math.isfinite(float(loss)) and grad.isfinite().all() and not grad[2].any() and not l[4].any()
    # the type's lowest values all along a row are as good as each other; large values leave no overflow
    for top in (torch.finfo(F32).min, torch.finfo(F32).max):
        even = torch.full_like(z, top).requires_grad_(True)
        _, l, stats = bnb.policy_loss(even, pick(acts), old, adv, **kw)
        want = -sum(math.log(n) for n in sizes)
        assert torch.allclose(l, torch.full_like(l, want), rtol=1e-5) and abs(float(stats[2]) + want) < 1e-4


def test_gradient_against_differences():
    import boost_and_broadside_b200 as bnb

    for sizes in ([3, 7, 2], [150], [1500]):
        z, acts, old, adv, ref = _inputs(12, sizes, F32)
        g = torch.Generator().manual_seed(1)
        way = torch.randn(z.shape, generator=g, dtype=torch.float64)
        many = sizes if len(sizes) > 1 else None
        kw = dict(ref=ref, sizes=sizes, clip=(0.2, 0.2), kl_coef=0.1, entropy_coef=0.05)
        at = lambda e: float(O.policy_loss(z.double() + e * way, acts, old, adv, **kw)[0])  # noqa: E731
        slope = (at(1e-6) - at(-1e-6)) / 2e-6
        x = z.to(DEV).requires_grad_(True)
        loss = bnb.policy_loss(x, (acts if many else acts[:, 0]).to(DEV), old.to(DEV), adv.to(DEV), ref_logprob=ref.to(DEV), sizes=many, kl_coef=0.1,
                               entropy_coef=0.05)[0]
        parts = torch.autograd.grad(loss, [x])[0].cpu().double() * way
        assert abs(float(parts.sum()) - slope) <= 2e-5 * float(parts.abs().sum())


def test_agrees_with_evaluate_action():
    import boost_and_broadside_b200 as bnb

    z, acts, old, adv, _ = (t.to(DEV) for t in _inputs(500, [3, 7, 2], F32))
    logprob, entropy = bnb.evaluate_action(z, acts)
    loss, l, stats = bnb.policy_loss(z, acts, old, adv, sizes=(3, 7, 2))
    assert torch.allclose(l, logprob, atol=1e-5) and abs(float(stats[2] - entropy.mean())) < 1e-5 and not loss.requires_grad


def test_captured_compiled_and_second_order():
    import boost_and_broadside_b200 as bnb

    for sizes in ([3, 7, 2], [3000]):
        many = sizes if len(sizes) > 1 else None
        z, acts, old, adv, ref = (t.to(DEV) for t in _inputs(30, sizes, BF16))
        acts = acts if many else acts[:, 0].contiguous()
        x = z.clone().requires_grad_(True)

        def call(x):
            return bnb.policy_loss(x, acts, old, adv, ref_logprob=ref, sizes=many, kl_coef=0.1, entropy_coef=0.01)

        def run():
            out = call(x)
            return *(t.detach() for t in out), *torch.autograd.grad(out[0] * 0.5, [x])

        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = run()
        with torch.no_grad():
            x.add_(torch.randn_like(x))
            adv.neg_()
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, run()))
        eager = call(x)
        compiled = torch.compile(call, fullgraph=True)(x)
        assert all(torch.equal(a, b) for a, b in zip(eager, compiled))
        got = [torch.autograd.grad(o[0] * 3.0, [x], retain_graph=o is eager)[0] for o in (eager, compiled, eager)]
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
        half, = torch.autograd.grad(eager[0] * 1.5, [x])
        assert torch.equal(half * 2, got[0])
        first, = torch.autograd.grad(call(x)[0], [x], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(first.float().sum(), [x])


def test_a_backward_captured_alone_repeats_itself():
    """The graph of an eager forward, its backward captured: every replay gives the same gradient."""
    import boost_and_broadside_b200 as bnb

    for dtype in (F32, BF16):
        z, acts, old, adv, _ = (t.to(DEV) for t in _inputs(8, [2048], dtype))
        x, a = z.clone().requires_grad_(True), acts[:, 0].contiguous()
        g = torch.full((), 0.5, device=DEV)
        stream = torch.cuda.Stream()          # autograd runs a backward on its forward's stream
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            loss = bnb.policy_loss(x, a, old, adv)[0]
            want = torch.autograd.grad(loss, [x], g, retain_graph=True)[0].clone()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, = torch.autograd.grad(loss, [x], g, retain_graph=True)
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_streams_and_hooks():
    import boost_and_broadside_b200 as bnb

    z, acts, old, adv, _ = (t.to(DEV) for t in _inputs(64, [4096], BF16))
    a = acts[:, 0].contiguous()
    x = z.clone().requires_grad_(True)
    want, = torch.autograd.grad(bnb.policy_loss(x, a, old, adv)[0], [x])
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got, = torch.autograd.grad(bnb.policy_loss(x, a, old, adv)[0], [x])
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(got, want)
    with torch.autograd.graph.save_on_cpu():
        loss = bnb.policy_loss(x, a, old, adv)[0]
    assert torch.equal(torch.autograd.grad(loss, [x])[0], want)
    loss = torch.utils.checkpoint.checkpoint(lambda v: bnb.policy_loss(v, a, old, adv)[0], x, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(loss, [x])[0], want)


def test_gradients_of_one_graph_again_and_again():
    """The first backward may hand out what the forward wrote; later ones, other factors and changed gradients do not see each other."""
    import boost_and_broadside_b200 as bnb

    for dtype, V in ((F32, 3001), (BF16, 2048), (F16, 2048), (BF16, 300)):
        z, acts, old, adv, ref = (t.to(DEV) for t in _inputs(20, [V], dtype))
        a, w = acts[:, 0].contiguous(), (torch.arange(20, device=DEV) % 3 + 0.5)
        kw = dict(ref_logprob=ref, kl_coef=0.1, entropy_coef=0.01, weights=w)
        x = z.clone().requires_grad_(True)
        grad = lambda loss, by: torch.autograd.grad(loss, [x], torch.tensor(by, device=DEV), retain_graph=True)[0]  # noqa: E731
        fresh = {by: grad(bnb.policy_loss(x, a, old, adv, **kw)[0], by).clone() for by in (1.0, 2.0, 0.0)}
        assert not fresh[0.0].any() and (dtype == F16 or torch.equal(fresh[1.0] * 2, fresh[2.0]))     # float16: numbers below its normal ones
        for by in (1.0, 2.0):
            assert torch.equal(grad(bnb.policy_loss(x, a, old, adv, grad_in_forward=False, **kw)[0], by), fresh[by])
        loss = bnb.policy_loss(x, a, old, adv, **kw)[0]
        for by in (1.0, 2.0, 1.0, 0.0, 1.0):
            got = grad(loss, by)
            assert torch.equal(got, fresh[by])
            got.add_(7)                                        # what was handed out is the caller's
        out = bnb.policy_loss(x, a, old, adv, **kw)
        (out[0] * 0.5 + bnb.policy_loss(x, a, old, adv, **kw)[0] * 0.5).backward()
        both = x.grad
        assert torch.allclose(both.float(), fresh[1.0].float(), rtol=2 * torch.finfo(dtype).eps, atol=1e-7)
        y = bnb.policy_loss(x, a, old, adv, **kw)[0]
        with torch.no_grad():
            x.add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            torch.autograd.grad(y, [x])
