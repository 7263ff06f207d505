"""The operators of an update's end together, behind the trunk: a head of ``linear`` layers on a trunk's sequence, ``policy_loss``, the backward through
both, ``AdamW`` over every parameter; eager and as one captured graph."""

import pytest
import torch

from oracle import update_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Head(torch.nn.Module):
    """Two layers with a residual one between them, as a user of the operators writes it."""

    def __init__(self, width: int, hidden: int, out: int) -> None:
        super().__init__()
        self.first, self.between, self.last = torch.nn.Linear(width, hidden), torch.nn.Linear(hidden, hidden), torch.nn.Linear(hidden, out)

    def forward(self, x):
        import boost_and_broadside_b200 as bnb

        h = bnb.linear(x, self.first.weight, self.first.bias, activation="gelu")
        h = bnb.linear(h, self.between.weight, self.between.bias, activation="silu", residual=h)
        return bnb.linear(h, self.last.weight, self.last.bias)


def _batch(T, B, N, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, B, N, D, generator=g).to(DEV)
    actions = torch.stack([torch.randint(n, (T, B, N), generator=g) for n in (3, 7, 2)], -1).to(DEV)
    old, adv = (-4 + 0.3 * torch.randn(T, B, N, generator=g)).to(DEV), torch.randn(T, B, N, generator=g).to(DEV)
    alive = (torch.rand(T, B, N, generator=g) < 0.8)
    alive[:, :, 0] = True
    return x, actions, old, adv, alive.to(DEV)


def test_head_gradients_through_loss_and_layers():
    """Against the formulas in 64 bits.  Float32: some hundred roundings along the longest chain, relative to a gradient's largest value."""
    import boost_and_broadside_b200 as bnb

    torch.manual_seed(0)
    head = Head(64, 96, 12).to(DEV)
    x, actions, old, adv, alive = _batch(2, 5, 3, 64)
    x.requires_grad_(True)
    loss, _, _ = bnb.policy_loss(head(x), actions, old, adv, weights=alive, sizes=(3, 7, 2), clip=(10.0, 10.0), entropy_coef=0.02)
    loss.backward()
    xl = x.detach().cpu().double().view(-1, 64).requires_grad_(True)
    w = [p.detach().cpu().double().requires_grad_(True) for p in head.parameters()]
    h = O.linear(xl, w[0], w[1], "gelu")
    h = O.linear(h, w[2], w[3], "silu", h)
    z = O.linear(h, w[4], w[5])
    flat = lambda t: t.cpu().reshape(30, *t.shape[3:])  # noqa: E731
    want, _, _ = O.policy_loss(z, flat(actions), flat(old), flat(adv), flat(alive), None, (3, 7, 2), (10.0, 10.0), 0.0, 0.02)
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5
    for got, v in zip([x.grad.view(-1, 64)] + [p.grad for p in head.parameters()], torch.autograd.grad(want, [xl, *w])):
        assert float((got.cpu().double() - v).abs().max()) <= 100 * 2.0 ** -23 * float(v.abs().max()) + 1e-9


@pytest.mark.parametrize("bits,bf16", [(32, False), (8, True)])
def test_updates_of_trunk_and_head(bits, bf16):
    import boost_and_broadside_b200 as bnb

    torch.manual_seed(1)
    T, B, N, D = 4, 3, 8, 128
    config = bnb.ModelConfig(d_model=D, n_heads=4, n_yemong_blocks=1)
    trunk, head = bnb.YemongTrunk(config).to(DEV), Head(D, 256, 12).to(DEV)
    params = [p for p in (*trunk.parameters(), *head.parameters())]
    x, actions, old, adv, alive = _batch(T, B, N, D)
    hidden = trunk.initial_hidden(B, N, torch.device(DEV))
    done = torch.zeros(T, B, dtype=torch.bool, device=DEV)
    done[1, 0] = True

    def update(trunk, head, opt):
        opt.zero_grad(set_to_none=True)
        with torch.autocast(DEV, dtype=torch.bfloat16, enabled=bf16):
            y, _ = trunk.sequence(x, alive, hidden, done)
            logits = head(y.bfloat16() if bf16 else y)
        loss, logprob, stats = bnb.policy_loss(logits, actions, old, adv, weights=alive, sizes=(3, 7, 2), entropy_coef=0.01)
        loss.backward()
        opt.step()
        return loss.detach(), stats

    twin_trunk, twin_head = bnb.YemongTrunk(config).to(DEV), Head(D, 256, 12).to(DEV)
    twin_trunk.load_state_dict(trunk.state_dict())
    twin_head.load_state_dict(head.state_dict())
    twins = [p for p in (*twin_trunk.parameters(), *twin_head.parameters())]
    make = lambda ps: bnb.AdamW(ps, lr=1e-3, max_norm=0.5, state_bits=bits, seed=5)  # noqa: E731
    opt, ref = make(params), make(twins)
    before = [p.detach().clone() for p in params]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        update(trunk, head, opt)                     # states and scratch exist before the capture
        update(twin_trunk, twin_head, ref)
    torch.cuda.synchronize()
    live = [p for p in params if p.grad is not None]
    assert len(live) >= len(list(head.parameters())) + 10
    assert all(p.grad.isfinite().all() for p in live) and sum(not torch.equal(a, b) for a, b in zip(before, params)) >= len(live) - 2
    assert float(opt.grad_norm) > 0
    graph = torch.cuda.CUDAGraph()
    opt.zero_grad(set_to_none=True)
    with torch.cuda.graph(graph, stream=stream):
        out = update(trunk, head, opt)
    with torch.cuda.stream(stream):
        for _ in range(3):
            graph.replay()
            want = update(twin_trunk, twin_head, ref)
    torch.cuda.synchronize()
    assert all(float(opt.state[p]["step"]) == 4 for p in live)
    # the trunk's parameter gradients are sums of atomics, whose order may differ: a part of a float32 step in each update
    assert float((out[0] - want[0]).abs()) <= 1e-3 and torch.allclose(out[1], want[1], atol=2e-3)
    assert all(p.isfinite().all() for p in params)
