"""Plain 64-bit implementations of the operators of an update's end, on the CPU (test infrastructure only), and first-order bounds of what a
float32 evaluation of the same formulas may be off by.  Every argument is taken to float64 first."""

from __future__ import annotations

import torch

U = 2.0 ** -24   # half a step of float32 relative to the value


def policy_loss(logits, actions, old, adv, weights=None, ref=None, sizes=None, clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0):
    """logits (R, V), actions (R, S) -> (loss, logprob (R), stats (4)); differentiable by autograd.  Rows of weight 0 are not looked at."""
    sizes = [logits.shape[1]] if sizes is None else list(sizes)
    w = torch.ones(logits.shape[0], dtype=torch.float64) if weights is None else weights.double()
    on = w != 0
    z = torch.where(on[:, None], logits.double(), 0.0)
    acts = torch.where(on[:, None], actions.reshape(-1, len(sizes)), 0)
    l, H, at = 0.0, 0.0, 0
    for i, n in enumerate(sizes):
        logp = torch.log_softmax(z[:, at:at + n], 1)
        l = l + logp.gather(1, acts[:, i:i + 1])[:, 0]
        p = logp.exp()
        H = H - torch.where(p > 0, p * torch.where(p > 0, logp, 0.0), 0.0).sum(1)
        at += n
    ratio, A = torch.exp(l - old.double()), adv.double()
    bound = ratio.clamp(1 - clip[0], 1 + clip[1]) * A
    surrogate = torch.min(ratio * A, bound)
    d = (ref.double() - l) if ref is not None else torch.zeros_like(l)
    k = torch.exp(d) - d - 1
    W = w.sum()
    mean = lambda v: (torch.where(on, v, 0.0) * w).sum() / W if W != 0 else w.sum() * 0  # noqa: E731
    beyond = ((ratio < 1 - clip[0]) | (ratio > 1 + clip[1])).double()
    stats = torch.stack([mean(surrogate), mean(k), mean(H), mean(beyond)])
    loss = -stats[0] + (kl_coef * stats[1] if kl_coef else 0.0) - entropy_coef * stats[2]
    return loss, torch.where(on, l, 0.0), stats


def policy_bounds(logits, actions, old, adv, weights=None, ref=None, sizes=None, clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0, scale=1.0,
                  additions=80):
    """What float32 results may be off by: (loss, logprob (R), stats (4), dlogits (R, V)), without the rounding of the results' own type.
    ``additions``: terms of a sum that are added one behind the other.  An exponential by the hardware's instruction is off by 2^-22 of its value,
    its argument t by three roundings."""
    sizes = [logits.shape[1]] if sizes is None else list(sizes)
    w = torch.ones(logits.shape[0], dtype=torch.float64) if weights is None else weights.double()
    on = w != 0
    z = torch.where(on[:, None], logits.double(), 0.0)
    acts = torch.where(on[:, None], actions.reshape(-1, len(sizes)), 0)
    parts, at = [], 0
    el = eH = l = H = 0.0
    for i, n in enumerate(sizes):
        part = z[:, at:at + n]
        m = part.amax(1, keepdim=True)
        t = (part - m).clamp(min=-1e4)
        e = t.exp()
        s = e.sum(1, keepdim=True)
        p = e / s
        a1, a2 = (p * t.abs()).sum(1, keepdim=True), (p * t * t).sum(1, keepdim=True)
        ds = U * (additions + 8 + 3 * a1)
        logs = s.log()
        h = logs + a1
        ta = t.gather(1, acts[:, i:i + 1])
        li = ta - logs
        el = el + ds + U * (ta.abs() + 2 * logs.abs() + 2 * li.abs())
        ehi = ds + U * (3 * logs.abs() + 2 * h.abs() + (additions + 8) * a1 + 3 * a2) + a1 * ds
        eH = eH + ehi
        lse = m + logs
        parts.append((at, n, p, t - logs, ds + U * (2 * lse.abs() + 2 * logs.abs()), h, ehi, acts[:, i:i + 1]))
        l, H = l + li, H + h
        at += n
    el = el[:, 0] + len(sizes) * U * l.abs()[:, 0]
    l, H, eH = l[:, 0], H[:, 0], eH[:, 0] + len(sizes) * U * H[:, 0].abs()
    o, A = old.double(), adv.double()
    ratio = torch.exp(l - o)
    er = ratio * (el + U * (4 + 2 * (l - o).abs()))
    es = A.abs() * (er + 2 * U * ratio.clamp(max=1 + clip[1]))
    d = ref.double() - l if ref is not None else torch.zeros_like(l)
    ek = (torch.exp(d) - 1).abs() * (el + U * d.abs()) + 3 * U * ((torch.exp(d) - 1).abs() + d.abs()) if ref is not None else torch.zeros_like(l)
    W = w.sum()
    mean = lambda v: (torch.where(on, v, 0.0) * w.abs()).sum() / W if W != 0 else W  # noqa: E731
    loss, _, stats = policy_loss(logits, actions, old, adv, weights, ref, sizes, clip, kl_coef, entropy_coef)
    estats = torch.stack([mean(es), mean(ek), mean(eH), torch.zeros((), dtype=torch.float64)]) + 2 * U * stats.abs()
    eloss = estats[0] + kl_coef * estats[1] + entropy_coef * estats[2] + 2 * U * loss.abs()
    share = (torch.where(on, w, 0.0) / W * scale).abs()
    active = (ratio * A <= ratio.clamp(1 - clip[0], 1 + clip[1]) * A).double()
    slope = -A * ratio * active - kl_coef * (torch.exp(d) - 1)
    eslope = A.abs() * er * active + U * (A * ratio).abs() * active + kl_coef * (torch.exp(d) * (el + U * d.abs()) + 3 * U * (torch.exp(d) - 1).abs())
    dl, edl = share * slope, share * (eslope + 6 * U * slope.abs())
    c2 = share * entropy_coef
    ez = torch.zeros_like(z)
    for at, n, p, t, elseb, h, ehi, act in parts:
        ep = p * (4 * U * t.abs() + 8 * U + elseb)
        c1 = c2[:, None] * h - dl[:, None]
        ec1 = c2[:, None] * (ehi + 8 * U * h.abs()) + edl[:, None] + U * c1.abs()
        v = ep * (c1.abs() + c2[:, None] * t.abs()) + p * (ec1 + c2[:, None] * (elseb + 8 * U * t.abs()) + 2 * U * (c1.abs() + c2[:, None] * t.abs()))
        hit = torch.zeros_like(p).scatter_(1, act, 1.0)
        ez[:, at:at + n] = v + hit * (edl + U * dl.abs())[:, None]
    return eloss, torch.where(on, el, 0.0), estats, torch.where(on[:, None], ez, 0.0)


def adamw(p, g, m, v, step, lr, betas, eps, decay, clip=1.0):
    """One step in 64 bits, m and v as they stand (the square of the root of 8-bit states): (p, m, v) behind it."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    t = step + 1
    g = g * clip
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    p = p * (1 - lr * decay) - lr / (1 - betas[0] ** t) * m / (v.sqrt() / (1 - betas[1] ** t) ** 0.5 + eps)
    return p, m, v


def adamw_bounds(p, g, m, v, step, lr, betas, eps, decay, clip=1.0):
    """What float32 results of the above may be off by: (p, m, v).  The factors count roundings: of the betas, of products and sums, of the clipping's
    factor (8, from a norm), of the bias corrections (6 each)."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    p1, m1, v1 = adamw(p, g, m, v, step, lr, betas, eps, decay, clip)
    t = step + 1
    em = U * (3 * (betas[0] * m).abs() + 12 * ((1 - betas[0]) * g * clip).abs())
    ev = U * (3 * betas[1] * v + 24 * (1 - betas[1]) * (g * clip) ** 2)
    r, root, rate = v1.sqrt(), (1 - betas[1] ** t) ** -0.5, lr / (1 - betas[0] ** t)
    er = torch.where(r > 0, ev / (2 * r.clamp(min=1e-300)), 0.0) + U * r
    d = r * root + eps
    ed = er * root + 8 * U * d
    q = rate * m1.abs() / d
    eq = rate * em / d + q * (ed / d + 12 * U)
    return eq + U * (4 * p.abs() + 2 * q + 2 * p1.abs()), em, ev


def noise(positions: torch.Tensor, seed: int, step: int) -> torch.Tensor:
    """The 20 random bits of 8-bit states: products and shifts of 32 bits."""
    low = lambda v: v & 0xFFFFFFFF  # noqa: E731
    h = low(low(positions + (positions >> 32) * 0x632BE5AB) * 0x9E3779B1 + seed * 0x5D2F63B9 + step * 0x3C6EF36B)
    h = low((h ^ (h >> 15)) * 0x6C8E944D)
    h = low((h ^ (h >> 13)) * 0x5B297A4D)
    return (h ^ (h >> 16)) >> 12


def linear(x, weight, bias=None, activation=None, residual=None):
    """act(x weight^T + bias) + residual; act is none, SiLU or erf GELU."""
    f = torch.nn.functional
    z = x.double() @ weight.double().t()
    z = z if bias is None else z + bias.double()
    y = {None: lambda v: v, "silu": f.silu, "gelu": f.gelu}[activation](z)
    return y if residual is None else y + residual.double()
