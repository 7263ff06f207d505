"""The operators behind the trunk in a policy update, over the sizes they are called at.

    linear  ``linear``: a matrix product with bias, activation and residual in its epilogue, with its gradients where trained
    policy  ``policy_loss``: the clipped policy loss with a KL term and the entropy, with the gradient of the logits
    adamw   ``AdamW``: one step over all parameter tensors, states in 32 or in 8 bits, gradients clipped by their global norm

Tensors of an optimizer are parts of one flat buffer each, every tensor from a multiple of 256 elements on, so that an update's results come
back as a few buffers; what stands between the tensors is zero and stays so.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256   # elements that share a scale of 8-bit states
CLIP = (0.2, 0.28)
KL, ENTROPY = 0.05, 0.01
LR, BETAS, EPS, DECAY, MAX_NORM, SEED = 3e-4, (0.9, 0.999), 1e-8, 0.01, 0.5, 20


def listed() -> list[dict]:
    return [
        # Two games being played: the first layer of a head on 16 ships.  Latency.
        _linear("linear_16x128x256", rows=16, width=128, out=256, act="gelu"),
        # One token through a wide layer: its weight has to be read.
        _linear("linear_1x4096x4096", rows=1, width=4096, out=4096, residual=True),
        # Odd sizes in float32, columns of a wider tensor, forward and backward.
        _linear("linear_train_301x522x130_fp32", rows=301, width=522, out=130, dtype="fp32", act="silu", residual=True, train=True, strided=True),
        # A minibatch of 8192 steps of 8 ships at the trunk's own width, forward and backward.
        _linear("linear_train_65536x128x512", rows=65536, width=128, out=512, act="gelu", train=True),
        # A wide layer, forward and backward.
        _linear("linear_train_8192x1024x4096", rows=8192, width=1024, out=4096, act="silu", residual=True, train=True),
        # A handful of steps of two games: latency.
        _policy("policy_16x12_fp32", rows=16, sizes="3,7,2", dtype="fp32", mask=True),
        # The minibatch of a recurrent update: 1024 environments of 8 ships, 32 steps, dead ships and forbidden actions among them.
        _policy("policy_262144x12", rows=262144, sizes="3,7,2", mask=True, forbidden=True),
        # Few rows of many actions, of an odd number, in float32, held near a reference policy.
        _policy("policy_1021x50021_fp32", rows=1021, sizes="50021", dtype="fp32", ref=True, mask=True),
        # Many rows of a vocabulary of actions, held near a reference policy.
        _policy("policy_4096x32768", rows=4096, sizes="32768", ref=True),
        # The policy's own parameters: many small tensors, clipped.  Latency.
        _adamw("adamw_99x1.7M", tensors=99, total=1_700_000, clip=True),
        # A larger policy with 8-bit states, tensors of odd sizes.
        _adamw("adamw_150x40M_8bit", tensors=150, total=40_000_001, bits=8),
        # The largest: memory alone counts.
        _adamw("adamw_64x120M", tensors=64, total=120_000_000),
    ]


def _linear(name, rows, width, out, dtype="bf16", act="none", bias=True, residual=False, train=False, strided=False):
    return dict(name=name, kind="linear", rows=rows, width=width, out=out, dtype=dtype, act=act, bias=bias, residual=residual, train=train,
                strided=strided)


def _policy(name, rows, sizes, dtype="bf16", ref=False, mask=False, forbidden=False, scale=1.0):
    return dict(name=name, kind="policy", rows=rows, sizes=sizes, dtype=dtype, ref=ref, mask=mask, forbidden=forbidden, scale=scale)


def _adamw(name, tensors, total, bits=32, dtype="fp32", clip=False):
    return dict(name=name, kind="adamw", tensors=tensors, total=total, bits=bits, dtype=dtype, clip=clip)


def draw(rng) -> dict:
    """One more case: an operator at random, its sizes over their logarithm, up to the work of its largest listed case."""

    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi) + 0.5))))))

    kind = rng.choice(("linear", "linear", "policy", "policy", "adamw"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "linear":
        width, out = log(1, 4200), log(1, 4200)
        if rng.random() < 0.6:
            width, out = (width + 7) // 8 * 8, (out + 7) // 8 * 8
        train = rng.random() < 0.6
        budget = (1 << 35) // (8 if dtype == "fp32" else 1)
        rows = log(1, max(1, min(65536, budget // (width * out))))
        case = _linear("", rows, width, out, dtype, rng.choice(("none", "silu", "gelu")), rng.random() < 0.8, rng.random() < 0.4, train,
                       rng.random() < 0.3)
    elif kind == "policy":
        if rng.random() < 0.4:
            sizes = rng.choice(("3,7,2", "3,7,2", ",".join(str(rng.randint(1, 40)) for _ in range(rng.randint(2, 8)))))
        else:
            sizes = str(log(2, 60000))
        rows = log(1, min(1 << 18, (1 << 27) // sum(int(n) for n in sizes.split(","))))
        scale = 2.0 * rows if dtype == "fp16" else rng.choice((1.0, 0.25, 3.0))   # a loss is scaled for float16, whose range ends at 6e-8
        case = _policy("", rows, sizes, dtype, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.3, scale)
    else:
        tensors = log(1, 200)
        total = log(tensors, 100_000_000)
        case = _adamw("", tensors, total, rng.choice((32, 8)), rng.choice(("fp32", "fp32", "bf16", "fp16")), rng.random() < 0.5)
    del case["name"]
    return case


# ----------------------------------------------------------------------------- inputs


def _sizes(case):
    return [int(n) for n in case["sizes"].split(",")]


def _tensors(case):
    """(first, elements) of each tensor in the flat buffers, and the buffers' size: sizes over a factor of some hundreds, odd ones among them."""
    rng = random.Random(case["tensors"])
    shares = [math.exp(rng.uniform(0, 6)) for _ in range(case["tensors"])]
    parts, at, left = [], 0, case["total"] - case["tensors"]
    whole = sum(shares)
    for i, v in enumerate(shares):
        n = 1 + (min(left, int((case["total"] - case["tensors"]) * v / whole)) if i + 1 < len(shares) else left)
        left -= n - 1
        parts.append((at, n))
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return parts, at


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case=dict(case))
    {"linear": _prepare_linear, "policy": _prepare_policy, "adamw": _prepare_adamw}[case["kind"]](case, s, g)
    return s


def _prepare_linear(case, s, g):
    M, K, N, dt = case["rows"], case["width"], case["out"], DTYPES[case["dtype"]]

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * by).to(dt)

    s["x"] = normal(M, K + 7)[:, 3:3 + K] if case["strided"] else normal(M, K)
    s["weight"] = normal(N, K, by=K ** -0.5)
    s["bias"] = normal(N, by=0.3) if case["bias"] else None
    s["residual"] = normal(M, N) if case["residual"] else None
    if case["train"]:
        s["dy"] = normal(M, N)
        if own:
            for k in _leaves(s):
                s[k] = s[k].requires_grad_(True)


def _leaves(s):
    return [k for k in ("x", "weight", "bias", "residual") if s[k] is not None]


def _prepare_policy(case, s, g):
    R, sizes, dt = case["rows"], _sizes(case), DTYPES[case["dtype"]]
    V, S = sum(sizes), len(sizes)
    z = (2.0 * torch.randn(R, V, device=DEV, generator=g)).to(dt)
    s["actions"] = torch.stack([torch.randint(n, (R,), device=DEV, generator=g) for n in sizes], -1)
    first = torch.tensor([sum(sizes[:i]) for i in range(S)], device=DEV)
    if case["forbidden"]:   # actions that the situation does not allow; those taken are allowed
        z = z.masked_fill((torch.rand(R, V, device=DEV, generator=g) < 0.2).scatter_(1, s["actions"] + first, False), -math.inf)
    s["slice_of"] = torch.repeat_interleave(torch.arange(S, device=DEV), torch.tensor(sizes, device=DEV))
    s["first"] = first
    # what the rollout recorded: the policy has moved a little since, and no ratio stands within 1e-3 of a border of the clipping
    moved = 0.2 * torch.randn(R, device=DEV, generator=g)
    for border in (1 - CLIP[0], 1 + CLIP[1]):
        moved = torch.where((torch.exp(moved) - border).abs() < 1e-3, moved + 0.01, moved)
    now = torch.zeros(R, device=DEV, dtype=torch.float64)
    for i, n in enumerate(sizes):
        part = z[:, int(first[i]):int(first[i]) + n]
        now += (part.gather(1, s["actions"][:, i:i + 1])[:, 0].float() - torch.logsumexp(part.float(), 1)).double()
    s["old"] = (now - moved).float()
    s["ref"] = (now + 0.3 * torch.randn(R, device=DEV, generator=g)).float() if case["ref"] else None
    s["advantages"] = torch.randn(R, device=DEV, generator=g)
    s["mask"] = None
    if case["mask"]:   # ships that are alive, one at least
        s["mask"] = torch.rand(R, device=DEV, generator=g) < 0.8
        s["mask"][0] = True
    s["scale"] = torch.full((), case["scale"], device=DEV)
    if S == 1:
        s["actions"] = s["actions"][:, 0].contiguous()
    s["logits"] = z.requires_grad_(True) if own else z


def _noise(positions: int, seed: int, step: int) -> torch.Tensor:
    """The random numbers of an 8-bit step: 20 bits for each position of the flat buffers, from 32-bit products and shifts of it, the seed and the step."""
    at = torch.arange(positions, device=DEV)
    h = ((at & 0xFFFFFFFF) + (at >> 32) * 0x632BE5AB) & 0xFFFFFFFF
    h = (h * 0x9E3779B1 + (seed * 0x5D2F63B9 + step * 0x3C6EF36B)) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x6C8E944D) & 0xFFFFFFFF
    h = h ^ (h >> 13)
    h = (h * 0x5B297A4D) & 0xFFFFFFFF
    return (h ^ (h >> 16)) >> 12


def _prepare_adamw(case, s, g):
    dt = DTYPES[case["dtype"]]
    parts, n = _tensors(case)
    inside = torch.zeros(n, device=DEV)
    for at, k in parts:
        inside[at:at + k] = 1

    def normal(by):
        return torch.randn(n, device=DEV, generator=g).mul_(by).mul_(inside)

    s["p"], s["g"] = normal(0.05).to(dt), normal(0.01).to(dt)
    s["steps"] = torch.full((len(parts),), 100.0, device=DEV)
    if case["bits"] == 8:
        s["m"] = normal(40.0).clamp_(-256, 256).to(torch.float8_e4m3fn)
        s["r"] = normal(40.0).abs_().clamp_(2 ** -6, 256).mul_(inside).to(torch.float8_e4m3fn)
        for k, low in (("m_scale", -16), ("r_scale", -14)):
            s[k] = torch.exp2(torch.randint(low, low + 4, (n // BLOCK,), device=DEV, generator=g).float())
        s["done"] = 100   # steps, for the plain form's random numbers
        names = {"exp_avg": "m", "exp_avg_scale": "m_scale", "exp_avg_sq_root": "r", "exp_avg_sq_root_scale": "r_scale"}
    else:
        s["m"], s["v"] = normal(0.005), normal(0.01).square_()
        names = {"exp_avg": "m", "exp_avg_sq": "v"}
    if own:
        import boost_and_broadside_b200 as bnb

        params = [torch.nn.Parameter(s["p"][at:at + k]) for at, k in parts]
        for p, (at, k) in zip(params, parts):
            p.grad = s["g"][at:at + k]
        s["optimizer"] = bnb.AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, max_norm=MAX_NORM if case["clip"] else None,
                                   state_bits=case["bits"], seed=SEED)
        for i, (p, (at, k)) in enumerate(zip(params, parts)):
            state = {name: s[b][at // BLOCK:(at + k + BLOCK - 1) // BLOCK] if name.endswith("scale") else s[b][at:at + k] for name, b in names.items()}
            s["optimizer"].state[p] = {"step": s["steps"][i], **state}


# ----------------------------------------------------------------------------- one pass


def run(s: dict):
    case = s["case"]
    if own:
        return _run_own(s, case)
    return {"linear": _plain_linear, "policy": _plain_policy, "adamw": _plain_adamw}[case["kind"]](s, case)


def _run_own(s, case):
    import boost_and_broadside_b200 as bnb

    if case["kind"] == "adamw":
        s["optimizer"].step()
        return _updated(s, case, s["optimizer"].grad_norm)
    if case["kind"] == "policy":
        loss, logprob, stats = bnb.policy_loss(s["logits"], s["actions"], s["old"], s["advantages"], weights=s["mask"], ref_logprob=s["ref"],
                                               sizes=_sizes(case) if "," in case["sizes"] else None, clip=CLIP, kl_coef=KL if case["ref"] else 0.0,
                                               entropy_coef=ENTROPY)
        return loss.detach(), logprob, stats, torch.autograd.grad(loss, [s["logits"]], s["scale"])[0]
    y = bnb.linear(s["x"], s["weight"], s["bias"], activation=None if case["act"] == "none" else case["act"], residual=s["residual"])
    if not case["train"]:
        return (y,)
    return y.detach(), *torch.autograd.grad(y, [s[k] for k in _leaves(s)], s["dy"])


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _activation(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "silu":
        sg = _sigmoid(z)
        return z * sg, sg * (1 + z * (1 - sg))
    cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def _plain_linear(s, case):
    dt = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y, slope = _activation(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if not case["train"]:
        return (y.to(dt),)
    dz = s["dy"].float() * slope
    grads = {"x": dz @ w, "weight": dz.t() @ x, "bias": dz.sum(0, dtype=torch.float64), "residual": s["dy"]}
    return y.to(dt), *(grads[k].to(dt) for k in _leaves(s))


def _plain_policy(s, case):
    z = s["logits"].float()
    R, S = z.shape[0], s["first"].numel()
    actions = s["actions"].reshape(R, S)
    many = S > 1
    of = s["slice_of"]
    one = (torch.arange(S, device=DEV)[None, :] == of[:, None]).float()   # (V, S): which logits are a slice's

    def over(v):   # sums over a slice
        return v @ one if many else v.sum(1, keepdim=True)

    def back(v):   # a slice's value at each of its logits
        return v[:, of] if many else v

    zero = torch.zeros((), device=DEV)
    top = torch.full((R, S), -math.inf, device=DEV).scatter_reduce(1, of.expand(R, -1), z, "amax") if many else z.amax(1, keepdim=True)
    t = z - back(top)
    e = torch.exp(t)
    norm = over(e)
    lse = torch.log(norm)
    te = torch.where(e == 0, zero, t * e)
    entropy = lse - over(te) / norm
    taken = actions + s["first"]
    logprob = (t.gather(1, taken) - lse).sum(1, dtype=torch.float64)
    weight = torch.ones(R, device=DEV) if s["mask"] is None else s["mask"].float()
    on = weight > 0
    total = weight.sum(dtype=torch.float64)
    ratio = torch.exp(logprob - s["old"].double())
    A = s["advantages"].double()
    held = ratio.clamp(1 - CLIP[0], 1 + CLIP[1])
    surrogate = torch.minimum(ratio * A, held * A)
    slope = torch.where(ratio * A <= held * A, -A * ratio, torch.zeros_like(A))
    kl = torch.zeros_like(A)
    if s["ref"] is not None:
        d = s["ref"].double() - logprob
        kl = torch.expm1(d) - d
        slope = slope - KL * torch.expm1(d)
    H = entropy.sum(1, dtype=torch.float64)
    outside = ((ratio < 1 - CLIP[0]) | (ratio > 1 + CLIP[1])).double()
    terms = torch.stack([surrogate, kl, H, outside], 1)
    stats = torch.where(on[:, None], terms * weight[:, None], torch.zeros_like(terms)).sum(0) / total
    loss = -stats[0] + (KL if case["ref"] else 0.0) * stats[1] - ENTROPY * stats[2]
    share = torch.where(on, weight.double() / total, torch.zeros_like(A)) * case["scale"]
    p = e / back(norm)
    dz = -p * (slope * share).float()[:, None]
    dz = dz.scatter_add(1, taken, (slope * share).float()[:, None].expand(-1, S))
    logp = t - back(lse)
    dz = dz + (ENTROPY * share).float()[:, None] * torch.where(p == 0, zero, p * (logp + back(entropy)))
    dz = torch.where(on[:, None], dz, zero)
    return loss.float(), torch.where(on, logprob, torch.zeros_like(A)).float(), stats.float(), dz.to(s["logits"].dtype)


def _updated(s, case, norm):
    states = ("m", "m_scale", "r", "r_scale") if case["bits"] == 8 else ("m", "v")
    return (s["p"], *(s[k] for k in states), s["steps"], *((norm,) if case["clip"] else ()))


def _plain_adamw(s, case):
    g = s["g"].float()
    norm = None
    if case["clip"]:
        norm = g.square().sum(dtype=torch.float64).sqrt()
        g = g * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0).float()
        norm = norm.float()
    s["steps"] += 1
    t = s["steps"][0].double()
    eight = case["bits"] == 8
    if eight:
        m = (s["m"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (s["r"].float().view(-1, BLOCK) * s["r_scale"][:, None]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + g * g * (1 - BETAS[1])
    r = v.sqrt()
    rate = (LR / (1 - BETAS[0] ** t)).float()
    root = (1 / (1 - BETAS[1] ** t).sqrt()).float()
    p = s["p"].float()
    p = p - p * (LR * DECAY) - rate * m / (r * root + EPS)
    s["p"].copy_(p)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return _updated(s, case, norm)
    s["done"] += 1
    for k, x in (("m", m), ("r", r)):
        most = x.view(-1, BLOCK).abs().amax(1)
        exponent = ((most.view(torch.int32) >> 23) - 7).clamp(min=1)
        s[k + "_scale"].copy_((exponent << 23).view(torch.float32))
        x = (x.view(-1, BLOCK) * ((254 - exponent) << 23).view(torch.float32)[:, None]).view(-1)   # by a power of two: exact
        if k == "r":
            up = (x.view(torch.int32) + _noise(x.numel(), SEED, s["done"]).to(torch.int32)) & ~0xFFFFF
            x = torch.where(x == 0, x, torch.where(x < 2 ** -6, torch.full_like(x, 2 ** -6), up.view(torch.float32)))
        s[k].copy_(x.to(torch.float8_e4m3fn))
    return _updated(s, case, norm)


# ----------------------------------------------------------------------------- what a pass cannot do without


def work(case: dict) -> dict:
    if case["kind"] == "adamw":
        n, es = case["total"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": n * 3 * es + (n * 16 if case["bits"] == 32 else n * 4 + n // BLOCK * 16), "flops": n * 15}
    es = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "policy":
        sizes = _sizes(case)
        R, V = case["rows"], sum(sizes)
        return {"bytes": 2 * R * V * es + R * (8 * len(sizes) + 12 + 4 * case["ref"] + case["mask"]), "flops": R * V * 12}
    M, K, N = case["rows"], case["width"], case["out"]
    b = M * K + K * N + M * N * (1 + case["residual"]) + N * case["bias"]
    if case["train"]:
        b += M * N + M * K + K * N + N * case["bias"]
    return {"bytes": b * es, "flops": 2 * M * K * N * (3 if case["train"] else 1)}


# ----------------------------------------------------------------------------- in 64 bits, from the definitions


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    return {"linear": _exact_linear, "policy": _exact_policy, "adamw": _exact_adamw}[case["kind"]](s, case)


def _exact_linear(s, case):
    f = torch.nn.functional
    names = _leaves(s)
    d = {k: None for k in ("bias", "residual")} | {k: s[k].detach().double().requires_grad_(case["train"]) for k in names}
    y = {"none": lambda v: v, "silu": f.silu, "gelu": f.gelu}[case["act"]](f.linear(d["x"], d["weight"], d["bias"]))
    if d["residual"] is not None:
        y = y + d["residual"]
    if not case["train"]:
        return (y,)
    return y.detach(), *torch.autograd.grad(y, [d[k] for k in names], s["dy"].double())


def _exact_policy(s, case):
    z = s["logits"].detach().double().requires_grad_(True)
    actions = s["actions"].reshape(z.shape[0], -1)
    logprob, H, at = 0.0, 0.0, 0
    for i, n in enumerate(_sizes(case)):
        logp = torch.log_softmax(z[:, at:at + n], 1)
        logprob = logprob + logp.gather(1, actions[:, i:i + 1])[:, 0]
        safe = logp.masked_fill(logp == -math.inf, 0.0)
        H = H - (logp.exp() * safe).sum(1)
        at += n
    weight = torch.ones_like(logprob) if s["mask"] is None else s["mask"].double()
    ratio, A = torch.exp(logprob - s["old"].double()), s["advantages"].double()
    surrogate = torch.min(ratio * A, torch.clip(ratio, 1 - CLIP[0], 1 + CLIP[1]) * A)
    d = s["ref"].double() - logprob if case["ref"] else torch.zeros_like(logprob)
    kl = torch.exp(d) - d - 1

    def mean(v):
        return (v * weight).sum() / weight.sum()

    loss = -mean(surrogate) + (KL * mean(kl) if case["ref"] else 0.0) - ENTROPY * mean(H)
    dz, = torch.autograd.grad(loss, [z], s["scale"].double())
    clipped = mean(((ratio < 1 - CLIP[0]) | (ratio > 1 + CLIP[1])).double())
    stats = torch.stack([mean(surrogate), mean(kl), mean(H), clipped])
    return loss.detach(), (logprob * (weight > 0)).detach(), stats.detach(), dz


def _exact_adamw(s, case):
    if case["bits"] == 8:
        first = s["m"].double() * s["m_scale"].double().repeat_interleave(BLOCK)
        second = (s["r"].double() * s["r_scale"].double().repeat_interleave(BLOCK)) ** 2
    else:
        first, second = s["m"].double(), s["v"].double()
    grad, p, t = s["g"].double(), s["p"].double(), 101
    norm = torch.linalg.vector_norm(grad)
    if case["clip"]:
        grad = grad * min(1.0, MAX_NORM / (float(norm) + 1e-6))
    first = torch.lerp(grad, first, BETAS[0])
    second = torch.lerp(grad ** 2, second, BETAS[1])
    p = p * (1 - LR * DECAY) - LR * (first / (1 - BETAS[0] ** t)) / (torch.sqrt(second / (1 - BETAS[1] ** t)) + EPS)
    last = (s["steps"].double() + 1, *((norm,) if case["clip"] else ()))
    if case["bits"] == 32:
        return (p, first, second, *last)
    scales = []
    for v in (first, second.sqrt()):
        most = v.view(-1, BLOCK).abs().amax(1)
        scales.append(torch.exp2(torch.floor(torch.log2(most)) - 7))
    m = (first.view(-1, BLOCK) / scales[0][:, None]).to(torch.float8_e4m3fn).double().view(-1)
    x = (second.sqrt().view(-1, BLOCK) / scales[1][:, None]).view(-1)
    step = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -6))) - 3)
    r = torch.floor(x / step + _noise(x.numel(), SEED, t).double() * 2.0 ** -20) * step
    r = torch.where(x == 0, torch.zeros_like(x), torch.where(x < 2.0 ** -6, torch.full_like(x, 2.0 ** -6), r))
    return (p, m, scales[0], r, scales[1], *last)
