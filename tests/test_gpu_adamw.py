"""``AdamW`` against its 64-bit implementation: many tensors and none, every type, states in 32 and 8 bits, clipping, layouts, captured steps, what is
saved and loaded.

Tolerances are first-order bounds of a float32 evaluation (``oracle.update_oracle.adamw_bounds``), elementwise, with half a step of the parameter's
type on top.  8-bit states have to be the codes that the formula gives wherever the value is further from where its rounding changes than those
bounds."""

import copy
import math

import pytest
import torch

from oracle import update_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HYPER = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def _within(got, want, bound, what):
    err = (got.detach().cpu().double() - want).abs()
    allowed = 1.1 * (bound + torch.finfo(got.dtype).eps / 2 * want.abs()) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
    assert bool((err <= allowed).all()), f"{what}: off by {float((err / allowed).max()):.2f} times what is allowed"


def _params(shapes, dtypes, seed=0):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.nn.Parameter((0.1 * torch.randn(s, generator=g)).to(d).to(DEV)) for s, d in zip(shapes, dtypes)]
    return ps, g


def _gradients(ps, g, by=0.02):
    for p in ps:
        p.grad = (by * torch.randn(p.shape, generator=g)).to(p.dtype).to(DEV)


def _value(state, name):
    """A state as the numbers it stands for, on the CPU in 64 bits."""
    v = state[name].detach().cpu().double()
    if name + "_scale" in state:
        v = (v.reshape(-1) * state[name + "_scale"].cpu().double().repeat_interleave(256)[:v.numel()]).view(v.shape)
    return v


SHAPES = [(7,), (1,), (256,), (255,), (257, 3), (0,), (2048,), (2049,), (4, 5, 6), (), (100, 130), (9000,)]
CASES = [
    # shapes, types, clipped
    (SHAPES, [F32] * 12, False),
    (SHAPES, [F32] * 12, True),
    (SHAPES, [BF16, F32, F16] * 4, True),
    ([(3, 3)] * 40, [F32] * 40, True),                     # more than the short list of tensors
    ([(5,), (300,)] * 200, [F32, BF16] * 200, True),       # more than the long one
    ([(3_000_001,), (17,)], [F32, F32], True),             # more chunks than CTAs
]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shapes,dtypes,clipped", CASES)
def test_adamw(shapes, dtypes, clipped, bits):
    import boost_and_broadside_b200 as bnb

    ps, g = _params(shapes, dtypes, seed=len(shapes))
    opt = bnb.AdamW(ps, **HYPER, max_norm=0.3 if clipped else None, state_bits=bits, seed=11)
    for step in range(3):
        _gradients(ps, g)
        before = [p.detach().cpu() for p in ps]
        names = ("exp_avg", "exp_avg_sq_root" if bits == 8 else "exp_avg_sq")
        old = [[_value(opt.state[p], n) if opt.state.get(p) else torch.zeros(p.shape, dtype=torch.float64) for n in names] for p in ps]
        kept = [p.grad.clone() for p in ps]
        opt.step()
        assert all(torch.equal(a, p.grad) for a, p in zip(kept, ps))
        clip = 1.0
        if clipped:
            norm = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
            assert abs(float(opt.grad_norm) - norm) <= 4 * O.U * norm
            clip = min(1.0, 0.3 / (norm + 1e-6))
        else:
            assert opt.grad_norm is None
        at = 0
        for p, was, (m, v) in zip(ps, before, old):
            st = opt.state[p]
            assert float(st["step"]) == step + 1
            v = v * v if bits == 8 else v
            args = (was, p.grad.cpu(), m, v, step, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"], clip)
            want, bound = O.adamw(*args), O.adamw_bounds(*args)
            _within(p, want[0], bound[0], "p")
            if bits == 32:
                _within(st["exp_avg"], want[1], bound[1], "m")
                _within(st["exp_avg_sq"], want[2], bound[2], "v")
            else:
                r = want[2].sqrt()
                er = torch.where(r > 0, bound[2] / (2 * r.clamp(min=1e-300)), 0.0) + 2 * O.U * r
                positions = torch.arange(p.numel()) + at
                _codes(st["exp_avg"], st["exp_avg_scale"], want[1], bound[1], None)
                _codes(st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"], r, er, O.noise(positions, 11, step + 1).double() / 2 ** 20)
            at += (p.numel() + 255) // 256 * 256


def _codes(codes, scale, want, bound, up):
    """Codes of e4m3 for values known within bounds: to nearest, or up where ``up`` says so."""
    n = want.numel()
    if n == 0:
        return
    x, e, c = want.reshape(-1), bound.reshape(-1), codes.cpu().double().reshape(-1)
    most = torch.nn.functional.pad(x.abs(), (0, -n % 256)).view(-1, 256).amax(1)
    exact = torch.exp2((torch.floor(torch.log2(most)) - 7).clamp(min=-126))
    s = scale.cpu().double()
    near = (torch.log2(most) - torch.round(torch.log2(most))).abs() < 1e-5      # at a power of two a rounding decides
    assert bool(((s == exact) | (near & ((s == 2 * exact) | (2 * s == exact)))).all())
    by = s.repeat_interleave(256)[:n]
    x, e = x / by, 1.1 * e / by + 1e-12
    if up is None:
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
        assert bool(((c - x).abs() <= step / 2 + e).all()), float(((c - x).abs() / step).max())
        return
    low = x < 2.0 ** -6
    step = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -6))) - 3)
    at = x / step + up
    sure = ((at - torch.round(at)).abs() > e / step + 1e-9) & ~low & (torch.log2(x.clamp(min=2.0 ** -6)).frac() > 1e-5)
    assert bool((c[sure] == (torch.floor(at) * step)[sure]).all())
    assert bool(((c - x).abs()[~low] <= (step + e)[~low]).all())
    assert bool((c[low] == torch.where(x[low] == 0, 0.0, 2.0 ** -6)).all())


def test_rounding_at_random_follows_small_changes():
    """A constant gradient: the root of the second moment arrives, where rounding to nearest would stop at a tenth of it.  It may end up to 7 %
    above: each step adds at most |change| x spacing of variance to v, in all root x spacing, and a spacing is at most an eighth.  The first moment is
    rounded to nearest: from below it stops where a tenth of what is missing is less than half a spacing of up to an eighth, 0.1 (g - m) < m / 16, so
    not below g / 1.625."""
    import boost_and_broadside_b200 as bnb

    p = torch.nn.Parameter(torch.zeros(8192, device=DEV))
    opt = bnb.AdamW([p], lr=1e-4, betas=(0.9, 0.999), state_bits=8, seed=3)
    p.grad = torch.full_like(p, 0.37)
    for _ in range(4000):
        opt.step()
    got = float(_value(opt.state[p], "exp_avg_sq_root").mean()) / (0.37 * (1 - 0.999 ** 4000) ** 0.5)
    assert 0.985 <= got <= 1.075, got
    assert 1 / 1.63 <= float(_value(opt.state[p], "exp_avg").mean()) / 0.37 <= 1.0


def test_groups_absent_gradients_and_repeated_steps():
    import boost_and_broadside_b200 as bnb

    ps, g = _params([(33,), (70, 3), (5,)], [F32] * 3)
    _gradients(ps, g)
    ps[2].grad = None
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for a, b in zip(twin, ps):
        a.grad = None if b.grad is None else b.grad.clone()
    make = lambda ps: bnb.AdamW([dict(params=ps[:1], lr=1e-2, betas=(0.5, 0.9)), dict(params=ps[1:], weight_decay=0.0)], **HYPER, max_norm=0.1, state_bits=8)  # noqa: E731
    a, b = make(ps), make(twin)
    for i in range(4):
        a.step()
        b.step()
        if i == 1:
            for o in (ps, twin):
                o[2].grad = torch.full_like(o[2], 0.5)
    for p, q in zip(ps, twin):
        assert torch.equal(p, q) and all(torch.equal(a.state[p][k].view(torch.uint8) if v.dtype == torch.float8_e4m3fn else a.state[p][k],
                                                     v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v) for k, v in b.state[q].items())
    assert [float(a.state[p]["step"]) for p in ps] == [4, 4, 2]
    none = torch.nn.Parameter(torch.zeros(3, device=DEV))
    o = bnb.AdamW([none])
    o.step()
    assert not o.state[none] and o.grad_norm is None
    a.zero_grad()
    was = ps[0].detach().clone()
    a.step()
    assert torch.equal(was, ps[0])


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits):
    """Clipped: the step is left out.  Not clipped: the element's state and value say so, no others of other blocks."""
    import boost_and_broadside_b200 as bnb

    for bad in (math.nan, math.inf):
        ps, g = _params([(1000,), (50,)], [F32] * 2)
        opt = bnb.AdamW(ps, **HYPER, max_norm=1.0, state_bits=bits)
        _gradients(ps, g)
        opt.step()
        kept = copy.deepcopy([(p.detach(), dict(opt.state[p])) for p in ps])
        ps[0].grad[700] = bad
        opt.step()
        assert not math.isfinite(float(opt.grad_norm))
        for p, (was, state) in zip(ps, kept):
            assert torch.equal(p, was)
            for k, v in state.items():
                assert torch.equal(opt.state[p][k].view(torch.uint8) if v.dtype == torch.float8_e4m3fn else opt.state[p][k], v.view(torch.uint8) if v.dtype == torch.float8_e4m3fn else v)
        opt = bnb.AdamW(ps, **HYPER, state_bits=bits)
        opt.step()
        assert ps[0][700].isnan() and not math.isfinite(float(opt.state[ps[0]]["exp_avg"][700]))
        assert ps[1].isfinite().all() and ps[0][:512].isfinite().all() and (bits == 8 or int((~ps[0].isfinite()).sum()) == 1)


def test_layouts():
    """Transposed parameters, gradients laid out otherwise, tensors off every boundary, an lr on the device."""
    import boost_and_broadside_b200 as bnb

    for bits in (32, 8):
        g = torch.Generator().manual_seed(1)
        flat = (0.1 * torch.randn(700, generator=g)).to(DEV)
        grads = (0.1 * torch.randn(700, generator=g)).to(DEV)
        dense = [torch.nn.Parameter(flat[1:301].clone()), torch.nn.Parameter(flat[303:643].clone())]
        odd = [torch.nn.Parameter(flat[1:301]), torch.nn.Parameter(flat[303:643].view(20, 17).t())]
        dense[0].grad, dense[1].grad = grads[1:301].clone(), grads[303:643].clone()
        odd[0].grad, odd[1].grad = grads[1:301], grads[303:643].view(20, 17).t().contiguous()
        one = bnb.AdamW(dense, **HYPER, state_bits=bits)
        two = bnb.AdamW(odd, **{**HYPER, "lr": torch.tensor(HYPER["lr"], device=DEV)}, state_bits=bits)
        edges = flat[[0, 301, 302, 643, 699]].clone()
        for _ in range(2):
            one.step()
            two.step()
        assert torch.equal(dense[0], odd[0]) and torch.equal(dense[1].view(20, 17).t(), odd[1]) and torch.equal(edges, flat[[0, 301, 302, 643, 699]])


def test_captured():
    import boost_and_broadside_b200 as bnb

    for bits in (32, 8):
        ps, g = _params([(300,), (65, 7), (4000,)], [F32, BF16, F32])
        twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        _gradients(ps, g)
        for a, b in zip(twin, ps):
            a.grad = b.grad.clone()
        lr = torch.tensor(1e-3, device=DEV)
        opt, ref = bnb.AdamW(ps, lr=lr, max_norm=0.5, state_bits=bits), bnb.AdamW(twin, lr=lr, max_norm=0.5, state_bits=bits)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            with pytest.raises(RuntimeError, match="before the capture"):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    opt.step()
            opt.step()
        torch.cuda.synchronize()
        ref.step()
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for graph in graphs:
            with torch.cuda.graph(graph, stream=stream):
                opt.step()
        for i in range(4):
            graphs[i % 2].replay()
            ref.step()
            torch.cuda.synchronize()
            lr.mul_(0.5)
            for a, b in zip(ps, twin):
                new = torch.randn_like(a)
                a.grad.copy_(new)
                b.grad.copy_(new)
        for a, b in zip(ps, twin):
            assert torch.equal(a, b) and float(opt.state[a]["step"]) == 5


def test_saved_and_loaded():
    import boost_and_broadside_b200 as bnb

    for bits in (32, 8):
        ps, g = _params([(300,), (65, 7), ()], [F32, BF16, F32])
        opt = bnb.AdamW(ps, **HYPER, max_norm=0.5, state_bits=bits, seed=4)
        _gradients(ps, g)
        opt.step()
        twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
        for a, b in zip(twin, ps):
            a.grad = b.grad.clone()
        other = bnb.AdamW(twin, lr=1.0, max_norm=0.5, state_bits=bits, seed=4)
        other.load_state_dict(copy.deepcopy(opt.state_dict()))
        for p in twin:
            assert other.state[p]["exp_avg"].dtype == (torch.float8_e4m3fn if bits == 8 else F32)
        opt.step()
        other.step()
        assert all(torch.equal(a, b) for a, b in zip(ps, twin))
        with pytest.raises(ValueError, match="does not fit"):
            bnb.AdamW(twin, state_bits=40 - bits).load_state_dict(opt.state_dict())
    both = copy.deepcopy((ps, opt))                          # a copy of parameters and optimizer goes on by itself
    for a, b in zip(both[0], ps):
        a.grad = b.grad.clone()
    both[1].step()
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip(both[0], ps)) and float(both[1].grad_norm) == float(opt.grad_norm)
    ps, g = _params([(300,), (65, 7)], [F32, F32])
    twin = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    _gradients(ps, g)
    for a, b in zip(twin, ps):
        a.grad = b.grad.clone()
    stock = torch.optim.AdamW(ps, **HYPER)
    stock.step()
    opt = bnb.AdamW(twin)
    for a, b in zip(twin, ps):
        a.data.copy_(b)
    opt.load_state_dict(stock.state_dict())
    stock.step()
    opt.step()
    for a, b in zip(ps, twin):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-8)


def test_another_stream_and_refusals():
    import boost_and_broadside_b200 as bnb

    ps, g = _params([(5000,)], [F32])
    twin = [torch.nn.Parameter(ps[0].detach().clone())]
    _gradients(ps, g)
    twin[0].grad = ps[0].grad.clone()
    one, two = bnb.AdamW(ps), bnb.AdamW(twin)
    one.step()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        two.step()
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(ps[0], twin[0])
    was = ps[0].detach().clone()
    good = one.state[ps[0]]["exp_avg"]
    for bad in (good[:10], good.double(), good.cpu()):
        one.state[ps[0]]["exp_avg"] = bad
        with pytest.raises(RuntimeError, match="exp_avg"):
            one.step()
    del one.state[ps[0]]["exp_avg"]
    with pytest.raises(RuntimeError, match="exp_avg"):
        one.step()
    one.state[ps[0]]["exp_avg"] = good
    strided = torch.nn.Parameter(torch.zeros(20, device=DEV)[::2])
    strided.grad = torch.zeros(10, device=DEV)
    with pytest.raises(ValueError, match="densely"):
        bnb.AdamW([strided]).step()
    whole = torch.zeros(300, device=DEV)
    shared = [torch.nn.Parameter(whole[:200]), torch.nn.Parameter(whole[199:])]
    shared[0].grad = torch.zeros(200, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        bnb.AdamW(shared).step()
    version = ps[0]._version
    assert torch.equal(was, ps[0]) and float(one.state[ps[0]]["step"]) == 1
    one.step()
    assert ps[0]._version > version
