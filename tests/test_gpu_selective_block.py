"""The operators together, as a temporal sublayer uses them: values, gradients of every parameter, single tokens against the sequence, padded
batches, replayed rollouts."""

import pytest
import torch
import torch.nn.functional as F

from oracle import sequence_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _block(D, N, seed=0):
    import boost_and_broadside_b200 as bnb

    torch.manual_seed(seed)
    block = bnb.SelectiveTemporalBlock(D, d_state=N)
    with torch.no_grad():
        for name, p in block.named_parameters():
            if p.dim() == 1 and "bias" not in name:
                p.add_(0.1 * torch.randn_like(p))
    return block


def _reference(block, p, x, h0, taps0, done=None, lengths=None):
    """The block in 64 bits from the definitions; p: its parameters by name; x (R, T, D)."""
    E, N = block.d_inner, block.d_state
    norm = lambda v, w: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + torch.finfo(torch.float32).eps) * w  # noqa: E731
    xt = x.transpose(0, 1)
    dt = None if done is None else done.transpose(0, 1)
    u, z = (norm(xt, p["norm1.weight"]) @ p["in_proj.weight"].T).split(E, -1)
    u, taps = O.causal_conv(u, p["conv.weight"][:, 0], p["conv.bias"], taps0, dt, lengths, "silu")
    d, B, C = (u @ p["x_proj.weight"].T).split([block.dt_rank, N, N], -1)
    y, h = O.selective_scan(u, d @ p["dt_proj.weight"].T, -torch.exp(p["A_log"]), B.unsqueeze(-2), C.unsqueeze(-2), p["D"], z, p["dt_proj.bias"], True, h0, dt, lengths)
    xt = xt + y @ p["out_proj.weight"].T
    n = norm(xt, p["norm2.weight"])
    return (xt + O.gated_mlp(n, p["gated_mlp.gate_proj.weight"], p["gated_mlp.up_proj.weight"], p["gated_mlp.down_proj.weight"])).transpose(0, 1), h, taps


@pytest.mark.parametrize("D,N,R,T", [(32, 16, 5, 12), (48, 4, 3, 70), (20, 9, 2, 33), (136, 16, 4, 9)])
def test_sequence_and_gradients(D, N, R, T):
    """float32 against 64 bits: a chain of eight float32 operators, each good to some 1e-6 of its result's size."""
    block = _block(D, N)
    g = torch.Generator().manual_seed(D)
    x, h0, taps0 = torch.randn(R, T, D, generator=g), 0.3 * torch.randn(R, 2 * D, N, generator=g), torch.randn(R, 3, 2 * D, generator=g)
    done = torch.rand(R, T, generator=g) < 0.15
    dy, dh, dt = torch.randn(R, T, D, generator=g), torch.randn(R, 2 * D, N, generator=g), torch.randn(R, 3, 2 * D, generator=g)
    names = [k for k, _ in block.named_parameters()]
    pd = {k: v.detach().double().requires_grad_(True) for k, v in block.named_parameters()}
    ins = [t.double().requires_grad_(True) for t in (x, h0, taps0)]
    want = _reference(block, pd, *ins, done)
    wg = torch.autograd.grad(want, [*ins, *pd.values()], [dy.double(), dh.double(), dt.double()])

    block = block.to(DEV)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, h0, taps0)]
    got = block.forward_sequence(*leaves, done.to(DEV))
    gg = torch.autograd.grad(got, [*leaves, *block.parameters()], [t.to(DEV) for t in (dy, dh, dt)])
    for name, a, b in zip(["out", "h", "taps", "x", "h0", "taps0", *names], [*got, *gg], [*want, *wg]):
        err = float((a.detach().cpu().double() - b.detach()).norm() / (b.detach().norm() + 1e-12))
        assert err <= 2e-5, (name, err)


def test_steps_are_the_sequence_and_replay():
    """A rollout of single tokens, captured once and replayed, moves the state as the sequence does."""
    D, N, R, T = 64, 16, 9, 6
    block = _block(D, N, 1).to(DEV)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(R, T, D, generator=g).to(DEV)
    done = (torch.rand(R, T, generator=g) < 0.3).to(DEV)
    h0, taps0 = 0.3 * torch.randn(R, 2 * D, N, generator=g).to(DEV), torch.randn(R, 3, 2 * D, generator=g).to(DEV)
    with torch.no_grad():
        want, wh, wt = block.forward_sequence(x, h0, taps0, done)
    xin, reset, h, taps = x[:, 0].clone(), torch.zeros(R, dtype=torch.bool, device=DEV), h0.clone(), taps0.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        block.step(xin, h, taps, reset)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = block.step(xin, h, taps, reset)
    h.copy_(h0)
    taps.copy_(taps0)
    for t in range(T):
        xin.copy_(x[:, t])
        reset.copy_(done[:, t - 1] if t else torch.zeros_like(reset))
        graph.replay()
        assert float((out - want[:, t]).abs().max()) <= 2e-5 * float(want.abs().max())
    assert float((h - wh).abs().max()) <= 2e-5 * float(wh.abs().max()) and float((taps - wt).abs().max()) <= 2e-5 * float(wt.abs().max())


def test_padded_prompts_then_tokens():
    """Prompts of different lengths in one batch give the states that each has alone, whatever stands behind their ends; a row without a
    prompt keeps its state."""
    D, N, T = 32, 8, 40
    block = _block(D, N, 2).to(DEV)
    g = torch.Generator().manual_seed(2)
    lengths = torch.tensor([40, 0, 1, 17, 39])
    R = len(lengths)
    x = torch.randn(R, T, D, generator=g)
    for r, n in enumerate(lengths.tolist()):
        x[r, n:] = float("nan")
    h0, taps0 = torch.randn(R, 2 * D, N, generator=g).to(DEV), torch.randn(R, 3, 2 * D, generator=g).to(DEV)
    with torch.no_grad():
        _, h, taps = block.forward_sequence(x.to(DEV), h0, taps0, lengths=lengths.to(DEV))
        for r, n in enumerate(lengths.tolist()):
            if n == 0:
                assert torch.equal(h[r], h0[r]) and torch.equal(taps[r], taps0[r])
                continue
            _, h1, t1 = block.forward_sequence(x[r:r + 1, :n].to(DEV), h0[r:r + 1], taps0[r:r + 1])
            assert float((h[r] - h1[0]).abs().max()) <= 2e-5 * float(h1.abs().max())
            assert float((taps[r] - t1[0]).abs().max()) <= 2e-5 * float(t1.abs().max())
    assert bool(torch.isfinite(h).all())


def test_under_autocast_and_compile():
    """bfloat16 inside autocast: within 16-bit rounding of the float32 block, forward and backward; one graph under the compiler."""
    D, N, R, T = 64, 16, 6, 20
    block = _block(D, N, 3).to(DEV)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(R, T, D, generator=g).to(DEV)
    h0, taps0 = block.initial_state(R, DEV)
    dy = torch.randn(R, T, D, generator=g).to(DEV)

    def run(fn, bf16):
        with torch.autocast(DEV, dtype=torch.bfloat16, enabled=bf16):
            y, h, taps = fn(x, h0, taps0)
        return y, torch.autograd.grad(y, list(block.parameters()), dy)

    y32, g32 = run(block.forward_sequence, False)
    y16, g16 = run(block.forward_sequence, True)
    assert float((y16.float() - y32).norm()) <= 2e-2 * float(y32.norm())
    for a, b in zip(g16, g32):
        assert float((a - b).norm()) <= 8e-2 * float(b.norm())
    yc, gc = run(torch.compile(block.forward_sequence, fullgraph=True), False)
    assert float((yc - y32).abs().max()) <= 1e-5 * float(y32.abs().max())
    for a, b in zip(gc, g32):
        assert float((a - b).norm()) <= 1e-4 * float(b.norm())


def test_refusals():
    import boost_and_broadside_b200 as bnb

    block = _block(32, 4).to(DEV)
    h, taps = block.initial_state(2, DEV)
    with pytest.raises(RuntimeError, match="shapes do not match"):
        block.forward_sequence(torch.zeros(3, 4, 32, device=DEV), h, taps)
    with pytest.raises(ValueError, match="d_state"):
        bnb.SelectiveTemporalBlock(32, d_state=65)
    u = torch.zeros(4, 2, 8, device=DEV)
    A, B = torch.zeros(8, 4, device=DEV), torch.zeros(4, 2, 4, device=DEV)
    with pytest.raises(RuntimeError, match="delta must be Float"):
        bnb.selective_scan(u, u.bfloat16(), A, B, B)
    with pytest.raises(RuntimeError, match="A must have shape"):
        bnb.selective_scan(u, u, torch.zeros(7, 4, device=DEV), B, B)
    with pytest.raises(ValueError, match="groups"):
        bnb.selective_scan(u, u, A, torch.zeros(4, 2, 3, 4, device=DEV), torch.zeros(4, 2, 3, 4, device=DEV))
    with pytest.raises(ValueError, match="states"):
        bnb.selective_scan(u, u, torch.zeros(8, 65, device=DEV), torch.zeros(4, 2, 65, device=DEV), torch.zeros(4, 2, 65, device=DEV))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        bnb.causal_conv(u.double(), torch.zeros(8, 4, device=DEV))
    with pytest.raises(ValueError, match="taps"):
        bnb.causal_conv(u, torch.zeros(8, 5, device=DEV))
    with pytest.raises(RuntimeError, match="done must have shape"):
        bnb.causal_conv(u, torch.zeros(8, 4, device=DEV), done=torch.zeros(2, 4, dtype=torch.bool, device=DEV))
    with pytest.raises(RuntimeError, match="is on cpu"):
        bnb.causal_conv(u, torch.zeros(8, 4))
    with pytest.raises(RuntimeError, match="contiguous"):
        bnb.selective_step(u[0], u[0], A, B[0], B[0], None, torch.zeros(2, 4, 8, device=DEV).transpose(1, 2))
    with pytest.raises(RuntimeError, match="weights must all be"):
        bnb.gated_mlp(u, torch.zeros(6, 8, device=DEV, dtype=torch.float16), torch.zeros(6, 8, device=DEV, dtype=torch.float16), torch.zeros(8, 6, device=DEV, dtype=torch.float16))
    # an operator that was refused leaves nothing behind: the next call works
    y, _ = bnb.causal_conv(u, torch.ones(8, 4, device=DEV))
    assert not F.relu(y).any()
