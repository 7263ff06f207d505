"""The operators of recurrent layers that this package offers outside its fixed trunk, over the sizes they are called at.

    conv       ``causal_conv``: the short depthwise convolution over time, whole sequences, with its gradients where trained
    conv_step  ``causal_conv_step``: one token a row, taps in place
    scan       ``selective_scan``: the selective state space recurrence over whole sequences, with its gradients where trained
    scan_step  ``selective_step``: one token a row, state in place
    gated      ``gated_mlp``: the gated feed-forward block, with its gradients where trained

Tensors are time-major like the trunk's: x (T, R, C), R rows that are sequences of their own (ships of all environments, or the
prompts of a batch).  ``done`` (T, R) ends an episode behind a step, ``lengths`` (R) the row.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # Prompts of different lengths in a batch-major program.
        _conv("conv_prompt_4x2047x1536", steps=2047, rows=4, width=1536, dtype="fp16", ragged=True, batch_major=True),
        # The minibatch of a recurrent update: 1024 environments of 8 ships, 32 steps, episode ends inside.
        _conv("conv_train_32x8192x256", steps=32, rows=8192, width=256, train=True, done=True),
        # Two games being played: latency.
        _conv_step("conv_step_16x256", rows=16, width=256, dtype="fp32"),
        # The rollout of a training run: 8192 environments of 8 ships.
        _conv_step("conv_step_65536x256", rows=65536, width=256, reset=True),
        # Two long prompts: few rows, many steps.
        _scan("scan_prompt_2x4093x1536", steps=4093, rows=2, width=1536, batch_major=True),
        # The minibatch above.
        _scan("scan_train_32x8192x256", steps=32, rows=8192, width=256, train=True, done=True),
        # Small odd sequences of different lengths trained in float32; two groups of channels share B and C.
        _scan("scan_train_301x3x522_fp32", steps=301, rows=3, width=522, states=11, groups=2, dtype="fp32", train=True, ragged=True),
        # Two games being played.
        _scan_step("scan_step_16x256", rows=16, width=256),
        # The rollout of a training run.
        _scan_step("scan_step_65536x256", rows=65536, width=256, reset=True),
        # Two games being played: the trunk's own width.
        _gated("gated_16x128x512", rows=16, width=128, hidden=512),
        # A minibatch of 8192 steps of 8 ships at the trunk's own width, forward and backward.
        _gated("gated_train_65536x128x512", rows=65536, width=128, hidden=512, train=True),
        # A wide block, forward and backward.
        _gated("gated_train_8192x1024x4096", rows=8192, width=1024, hidden=4096, act="silu", train=True),
    ]


def _conv(name, steps, rows, width, taps=4, dtype="bf16", act="silu", train=False, done=False, ragged=False, batch_major=False):
    return dict(name=name, kind="conv", steps=steps, rows=rows, width=width, taps=taps, dtype=dtype, act=act, train=train, done=done,
                ragged=ragged, batch_major=batch_major)


def _conv_step(name, rows, width, taps=4, dtype="bf16", act="silu", reset=False):
    return dict(name=name, kind="conv_step", rows=rows, width=width, taps=taps, dtype=dtype, act=act, reset=reset)


def _scan(name, steps, rows, width, states=16, groups=1, dtype="bf16", train=False, done=False, ragged=False, batch_major=False):
    return dict(name=name, kind="scan", steps=steps, rows=rows, width=width, states=states, groups=groups, dtype=dtype, train=train,
                done=done, ragged=ragged, batch_major=batch_major)


def _scan_step(name, rows, width, states=16, groups=1, dtype="bf16", reset=False):
    return dict(name=name, kind="scan_step", rows=rows, width=width, states=states, groups=groups, dtype=dtype, reset=reset)


def _gated(name, rows, width, hidden, dtype="bf16", act="gelu", train=False):
    return dict(name=name, kind="gated", rows=rows, width=width, hidden=hidden, dtype=dtype, act=act, train=train)


def draw(rng) -> dict:
    """One more case: an operator at random, its sizes over their logarithm, up to the work of its largest listed case."""

    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi) + 0.5))))))

    kind = rng.choice(("conv", "conv_step", "scan", "scan", "scan_step", "gated", "gated"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    width = log(17, 2100)
    if rng.random() < 0.6:
        width = (width + 7) // 8 * 8
    if kind == "conv":
        steps = log(1, 4096)
        case = _conv("", steps, log(1, max(1, (1 << 25) // (steps * width))), width, rng.randint(2, 4), dtype, rng.choice(("silu", "none")),
                     rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.4, rng.random() < 0.5)
    elif kind == "conv_step":
        case = _conv_step("", log(1, (1 << 23) // width), width, rng.randint(2, 4), dtype, rng.choice(("silu", "none")), rng.random() < 0.5)
    elif kind == "gated":
        hidden = log(width, 4 * width)
        if rng.random() < 0.6:
            hidden = (hidden + 7) // 8 * 8
        budget = (1 << 33) if dtype == "fp32" else (1 << 34)
        case = _gated("", log(1, min(65536, budget // (width * hidden))), width, hidden, dtype, rng.choice(("gelu", "silu")), rng.random() < 0.7)
    else:
        groups = rng.choice((1, 1, 2, 4))
        width = (width + groups - 1) // groups * groups
        states = rng.choice((16, 16, 16, 8, 4, rng.randint(1, 32), 32, 64))
        if kind == "scan":
            train = rng.random() < 0.6
            steps = log(1, 1024 if train else 4096)
            cells = (1 << 27) // (steps * width * states)
            case = _scan("", steps, log(1, max(1, cells)), width, states, groups, dtype, train, rng.random() < 0.4, rng.random() < 0.4,
                         rng.random() < 0.5)
        else:
            case = _scan_step("", log(1, (1 << 26) // (width * states)), width, states, groups, dtype, rng.random() < 0.5)
    del case["name"]
    return case


# ----------------------------------------------------------------------------- inputs


def _lengths(case):
    """Row r of a ragged batch: between half the steps and all of them; some rows of larger batches are empty."""
    T, R = case["steps"], case["rows"]
    r = torch.arange(R)
    n = T - (r * 37) % (T // 2 + 1)
    n[r % 11 == 7] = 0
    return n.to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, device=DEV, generator=g)

    def rows_of(*widths):
        """Column ranges of one projection's output, as a layer slices it: (T, R, width) each, strided."""
        T, R = case["steps"], case["rows"]
        big = normal(*((R, T) if case["batch_major"] else (T, R)), sum(widths))
        if case["batch_major"]:
            big = big.transpose(0, 1)
        return list(big.split(list(widths), dim=-1))

    s = dict(case=dict(case))
    kind, C = case["kind"], case["width"]
    if kind in ("conv", "conv_step"):
        R, K = case["rows"], case["taps"]
        s["weight"] = normal(C, K, dtype=torch.float32) * (0.6 / K ** 0.5)
        s["bias"] = normal(C, dtype=torch.float32) * 0.1
        s["state"] = normal(R, K - 1, C, dtype=torch.float32)
        if kind == "conv":
            s["x"] = rows_of(C, C)[0]
    elif kind in ("scan", "scan_step"):
        R, N, G = case["rows"], case["states"], case["groups"]
        s["A"] = -torch.arange(1, N + 1, device=DEV, dtype=torch.float32).expand(C, N) * (1 + 0.05 * normal(C, N, dtype=torch.float32)).abs()
        s["D"] = 1 + 0.1 * normal(C, dtype=torch.float32)
        rate = torch.exp(uniform(C) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))   # steps of 0.001 to 0.1 at a zero input
        s["delta_bias"] = rate + torch.log(-torch.expm1(-rate))
        s["state"] = 0.5 * normal(R, C, N, dtype=torch.float32)
        if kind == "scan":
            s["u"], s["z"] = rows_of(C, C)
            s["delta"], = rows_of(C)
            _, b, c = rows_of(8, G * N, G * N)
            s["B"], s["C"] = b.unflatten(-1, (G, N)), c.unflatten(-1, (G, N))
        else:
            s["u"], s["z"] = normal(R, 2 * C).split(C, dim=-1)
            s["delta"] = normal(R, C)
            _, b, c = normal(R, 8 + 2 * G * N).split([8, G * N, G * N], dim=-1)
            s["B"], s["C"] = b.unflatten(-1, (G, N)), c.unflatten(-1, (G, N))
    else:
        M, F = case["rows"], case["hidden"]
        s["x"] = normal(M, C)
        s["gate_w"] = normal(F, C, dtype=torch.float32).mul_(C ** -0.5).to(dt)
        s["up_w"] = normal(F, C, dtype=torch.float32).mul_(C ** -0.5).to(dt)
        s["down_w"] = normal(C, F, dtype=torch.float32).mul_(F ** -0.5).to(dt)
    if kind == "conv_step":
        s["x"] = normal(case["rows"], C)
    s["done"] = uniform(case["steps"], case["rows"]) < 0.03 if case.get("done") else None
    s["reset"] = uniform(case["rows"]) < 0.03 if case.get("reset") else None
    s["lengths"] = _lengths(case).to(DEV) if case.get("ragged") else None
    if case.get("train"):
        s["dy"] = normal(*((case["rows"], C) if kind == "gated" else (case["steps"], case["rows"], C)))
        if kind != "gated":
            s["dstate"] = normal(*s["state"].shape, dtype=torch.float32)
        if own:
            for k in _leaves(case):
                s[k].requires_grad_(True)
    return s


def _leaves(case):
    """What the gradients of a trained case are taken for, in the order they are returned."""
    return {"conv": ("x", "weight", "bias", "state"),
            "scan": ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state"),
            "gated": ("x", "gate_w", "up_w", "down_w")}[case["kind"]]


# ----------------------------------------------------------------------------- one pass


def run(s: dict):
    case = s["case"]
    if own:
        return _run_own(s, case)
    return {"conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan, "scan_step": _plain_scan_step,
            "gated": _plain_gated}[case["kind"]](s, case)


def _run_own(s, case):
    import boost_and_broadside_b200 as bnb

    kind = case["kind"]
    act = None if case.get("act") == "none" else case.get("act")
    if kind == "conv_step":
        y = bnb.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], reset=s["reset"], activation=act)
        return y, s["state"]
    if kind == "scan_step":
        y = bnb.selective_step(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], s["state"], z=s["z"], delta_bias=s["delta_bias"],
                               softplus=True, reset=s["reset"])
        return y, s["state"]
    if kind == "conv":
        outs = bnb.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], done=s["done"], lengths=s["lengths"], activation=act)
    elif kind == "scan":
        outs = bnb.selective_scan(s["u"], s["delta"], s["A"], s["B"], s["C"], s["D"], z=s["z"], delta_bias=s["delta_bias"], softplus=True,
                                  state=s["state"], done=s["done"], lengths=s["lengths"])
    else:
        outs = (bnb.gated_mlp(s["x"], s["gate_w"], s["up_w"], s["down_w"], activation=act),)
    if not case["train"]:
        return outs
    given = (s["dy"],) if kind == "gated" else (s["dy"], s["dstate"])
    return *(o.detach() for o in outs), *torch.autograd.grad(outs, [s[k] for k in _leaves(case)], given)


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _episodes(case, done):
    """(T, R) number of episodes that ended before each step."""
    T, R = case["steps"], case["rows"]
    n = torch.zeros(T, R, dtype=torch.int32, device=DEV)
    if done is not None and T > 1:
        n[1:] = torch.cumsum(done[:-1].int(), 0)
    return n


def _alive_steps(case, lengths):
    """(T, R, 1) whether a step is before its row's end."""
    T = case["steps"]
    return None if lengths is None else (torch.arange(T, device=DEV)[:, None] < lengths[None, :])[..., None]


def _plain_conv(s, case):
    T, R, C, K = case["steps"], case["rows"], case["width"], case["taps"]
    dt = s["x"].dtype
    live = _alive_steps(case, s["lengths"])
    x = s["x"].float()
    if live is not None:
        x = torch.where(live, x, torch.zeros_like(x))
    padded = torch.cat([s["state"].transpose(0, 1), x], 0)                    # step t stands at t + K - 1
    ended = torch.cat([torch.zeros(K - 1, R, dtype=torch.int32, device=DEV), _episodes(case, s["done"])], 0)
    same = [(ended[K - 1 - j:K - 1 - j + T] == ended[K - 1:])[..., None] for j in range(K)]   # the step j before, in this episode?
    w = s["weight"]
    pre = s["bias"] + torch.zeros_like(x)
    for j in range(K):
        pre = pre + w[:, K - 1 - j] * torch.where(same[j], padded[K - 1 - j:K - 1 - j + T], torch.zeros((), device=DEV))
    silu = case["act"] == "silu"
    y = pre * _sigmoid(pre) if silu else pre
    if live is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    # taps behind the last step: those of its own episode
    n = (torch.full((R,), T, device=DEV) if s["lengths"] is None else s["lengths"]).long()
    at = torch.stack([n + i for i in range(K - 1)])                            # their rows in `padded`
    last = ended.gather(0, (n + K - 2)[None].clamp(min=0))
    keep = (ended.gather(0, at) == last)[..., None]
    taps = torch.where(keep, padded.gather(0, at[..., None].expand(-1, -1, C)), torch.zeros((), device=DEV))
    outs = (y.to(dt), taps.transpose(0, 1).contiguous())
    if not case["train"]:
        return outs
    dpre = s["dy"].float()
    if live is not None:
        dpre = torch.where(live, dpre, torch.zeros_like(dpre))
    if silu:
        sg = _sigmoid(pre)
        dpre = dpre * (sg * (1 + pre * (1 - sg)))
    dpad = torch.zeros_like(padded)
    dw = torch.zeros_like(w)
    for j in range(K):
        lag = padded[K - 1 - j:K - 1 - j + T]
        dpad[K - 1 - j:K - 1 - j + T] += torch.where(same[j], dpre * w[:, K - 1 - j], torch.zeros((), device=DEV))
        dw[:, K - 1 - j] = torch.where(same[j], dpre * lag, torch.zeros((), device=DEV)).sum((0, 1), dtype=torch.float64).float()
    dtaps = torch.where(keep, s["dstate"].transpose(0, 1), torch.zeros((), device=DEV))
    dpad.scatter_add_(0, at[..., None].expand(-1, -1, C), dtaps)
    db = dpre.sum((0, 1), dtype=torch.float64).float()
    return *outs, dpad[K - 1:].to(dt), dw, db, dpad[:K - 1].transpose(0, 1).contiguous()


def _plain_conv_step(s, case):
    state, x = s["state"], s["x"].float()
    if s["reset"] is not None:
        state = torch.where(s["reset"][:, None, None], torch.zeros_like(state), state)
    window = torch.cat([state, x[:, None]], 1)
    pre = s["bias"] + (window * s["weight"].t()).sum(1)
    y = pre * _sigmoid(pre) if case["act"] == "silu" else pre
    s["state"].copy_(window[:, 1:])
    return y.to(s["x"].dtype), s["state"]


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20))))


def _shared(v, case):
    """(..., G, N) of the groups to (..., C, N) of the channels, in float32."""
    return v.float().repeat_interleave(case["width"] // case["groups"], dim=-2)


def _plain_scan(s, case):
    T, R = case["steps"], case["rows"]
    A, D = s["A"], s["D"]
    dt = s["u"].dtype
    live, done = _alive_steps(case, s["lengths"]), s["done"]
    zero = torch.zeros((), device=DEV)
    raw = [s["delta"][t].float() + s["delta_bias"] for t in range(T)]
    keeps = case["train"]
    hs, ys = [], []
    h = s["state"].float().clone()
    out = torch.empty(T, R, case["width"], dtype=dt, device=DEV)
    for t in range(T):
        held = h
        if t > 0 and done is not None:
            h = torch.where(done[t - 1][:, None, None], zero, h)
        p, u = _softplus(raw[t]), s["u"][t].float()
        new = torch.exp(p[..., None] * A) * h + (p * u)[..., None] * _shared(s["B"][t], case)
        y = (new * _shared(s["C"][t], case)).sum(-1) + D * u
        z = s["z"][t].float()
        o = y * z * _sigmoid(z)
        if keeps:
            hs.append(h)
            ys.append(y)
        if live is not None:
            new = torch.where(live[t][..., None], new, held)
            o = torch.where(live[t], o, zero)
        h = new
        out[t] = o.to(dt)
    if not keeps:
        return out, h
    du, ddelta, dz = (torch.empty(T, R, case["width"], dtype=dt, device=DEV) for _ in range(3))
    dB, dC = (torch.empty(s["B"].shape, dtype=dt, device=DEV) for _ in range(2))
    dA, dD, dbias = (torch.zeros(v.shape, dtype=torch.float64, device=DEV) for v in (A, D, s["delta_bias"]))
    G, Cg = case["groups"], case["width"] // case["groups"]
    carry = s["dstate"]                       # gradient of the state behind step t
    for t in range(T - 1, -1, -1):
        p, u, z = _softplus(raw[t]), s["u"][t].float(), s["z"][t].float()
        Bt, Ct = _shared(s["B"][t], case), _shared(s["C"][t], case)
        a = torch.exp(p[..., None] * A)
        before = hs[t]
        new = a * before + (p * u)[..., None] * Bt
        do = s["dy"][t].float()
        sg = _sigmoid(z)
        dy = do * z * sg
        dzt = do * ys[t] * sg * (1 + z * (1 - sg))
        dh = carry + dy[..., None] * Ct
        dCt = (dy[..., None] * new).unflatten(1, (G, Cg)).sum(2)
        dBt = (dh * (p * u)[..., None]).unflatten(1, (G, Cg)).sum(2)
        dhB = (dh * Bt).sum(-1)
        g = dh * a * before
        dp = (g * A).sum(-1) + dhB * u
        dut = dhB * p + dy * D
        draw_t = dp * torch.where(raw[t] > 20, torch.ones_like(p), _sigmoid(raw[t]))
        back = dh * a
        if t > 0 and done is not None:
            back = torch.where(done[t - 1][:, None, None], zero, back)
        dAt, dDt = g * p[..., None], dy * u
        if live is not None:
            lt = live[t]
            dut, draw_t, dzt, dDt = (torch.where(lt, v, zero) for v in (dut, draw_t, dzt, dDt))
            dAt, dBt, dCt = (torch.where(lt[..., None], v, zero) for v in (dAt, dBt, dCt))
            back = torch.where(lt[..., None], back, carry)
        dA += dAt.sum(0)
        dD += dDt.sum(0)
        dbias += draw_t.sum(0)
        du[t], ddelta[t], dz[t], dB[t], dC[t] = dut.to(dt), draw_t.to(dt), dzt.to(dt), dBt.to(dt), dCt.to(dt)
        carry = back
        hs[t] = ys[t] = None
    return out, h, du, ddelta, dA.float(), dB, dC, dD.float(), dz, dbias.float(), carry


def _plain_scan_step(s, case):
    h = s["state"]
    if s["reset"] is not None:
        h = torch.where(s["reset"][:, None, None], torch.zeros_like(h), h)
    p, u, z = _softplus(s["delta"].float() + s["delta_bias"]), s["u"].float(), s["z"].float()
    new = torch.exp(p[..., None] * s["A"]) * h + (p * u)[..., None] * _shared(s["B"], case)
    y = (new * _shared(s["C"], case)).sum(-1) + s["D"] * u
    s["state"].copy_(new)
    return (y * z * _sigmoid(z)).to(s["u"].dtype), s["state"]


def _activation(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        sg = _sigmoid(g)
        return g * sg, sg * (1 + g * (1 - sg))
    cdf = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _plain_gated(s, case):
    dt = s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "gate_w", "up_w", "down_w"))
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _activation(g, case["act"])
    h = a * u
    y = (h @ wd.t()).to(dt)
    if not case["train"]:
        return (y,)
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    return y, (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt), (dy.t() @ h).to(dt)


# ----------------------------------------------------------------------------- what a pass cannot do without


def work(case: dict) -> dict:
    es = 4 if case["dtype"] == "fp32" else 2
    kind, C, R = case["kind"], case["width"], case["rows"]
    train = case.get("train", False)
    if kind == "gated":
        F = case["hidden"]
        weights, rows = 3 * C * F, R * C
        return {"bytes": es * (weights * (2 if train else 1) + rows * (4 if train else 2)), "flops": 2 * R * weights * (3 if train else 1)}
    if kind == "conv_step":
        K = case["taps"]
        return {"bytes": 2 * R * C * es + 8 * R * (K - 1) * C + 4 * C * (K + 1), "flops": R * C * (2 * K + 4)}
    if kind == "scan_step":
        N, G = case["states"], case["groups"]
        return {"bytes": 4 * R * C * es + 2 * R * G * N * es + 8 * R * C * N + 4 * C * (N + 2), "flops": R * C * (7 * N + 12)}
    T = case["steps"]
    read = int(_lengths(case).sum()) if case["ragged"] else T * R    # steps that are looked at; all are written
    if kind == "conv":
        K = case["taps"]
        b = es * C * (read + T * R) + 8 * R * (K - 1) * C + 4 * C * (K + 1)
        f = read * C * (2 * K + 4)
        if train:   # dy read, dx written; dstate, weights and their gradients
            b += es * C * (read + T * R) + 8 * R * (K - 1) * C + 4 * C * (K + 1)
            f += read * C * (6 * K + 8)
        return {"bytes": b, "flops": f}
    N, G = case["states"], case["groups"]
    b = es * (C * (3 * read + T * R) + 2 * G * N * read) + 8 * R * C * N + 4 * C * (N + 2)
    f = read * C * (7 * N + 12)
    if train:
        b += es * (C * (read + 3 * T * R) + 2 * G * N * T * R) + 8 * R * C * N + 4 * C * (N + 2)
        f += read * C * (18 * N + 20)
    return {"bytes": b, "flops": f}


# ----------------------------------------------------------------------------- in 64 bits, from the definitions


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    d = {k: (v.detach().double() if torch.is_tensor(v) and v.is_floating_point() else v) for k, v in s.items()}
    del s
    kind = case["kind"]
    if kind == "gated":
        return _exact_gated(d, case)
    if kind in ("conv_step", "scan_step"):   # a sequence of one step whose state is cleared first
        one = dict(case, steps=1, train=False)
        seq = {k: v[None] for k, v in d.items() if k in ("x", "u", "delta", "B", "C", "z")}
        if d["reset"] is not None:
            d["state"] = d["state"].masked_fill(d["reset"][:, None, None], 0)
        y, state = _exact_rows(one, {**d, **seq, "lengths": None, "done": None})
        return y[0], state
    if not case["train"]:
        return _exact_rows(case, d)
    # gradients by automatic differentiation, a block of rows at a time
    names = _leaves(case)
    per_row = {"x": 1, "u": 1, "delta": 1, "B": 1, "C": 1, "z": 1, "dy": 1, "done": 1, "state": 0, "dstate": 0, "lengths": 0}
    cells = case["steps"] * case["width"] * case.get("states", 1)
    block = max(1, (1 << 27) // cells)
    parts, totals = [], {}
    for r in range(0, case["rows"], block):
        rows = slice(r, min(r + block, case["rows"]))
        part = {k: (v if k not in per_row or v is None else v[:, rows] if per_row[k] else v[rows]) for k, v in d.items()}
        leaves = [part[k].detach().clone().requires_grad_(True) for k in names]
        y, state = _exact_rows(case, {**part, **dict(zip(names, leaves))})
        grads = torch.autograd.grad([y, state], leaves, [part["dy"], part["dstate"]])
        parts.append([y.detach(), state.detach(), *(g if k in per_row else None for k, g in zip(names, grads))])
        for k, g in zip(names, grads):
            if k not in per_row:
                totals[k] = totals.get(k, 0) + g
    joined = []
    for i, k in enumerate(("dy", "state", *names)):
        joined.append(totals[k] if k not in per_row else torch.cat([p[i] for p in parts], per_row[k]))
    return tuple(joined)


def _exact_rows(case, d):
    return _exact_conv(case, d) if case["kind"].startswith("conv") else _exact_scan(case, d)


def _exact_conv(case, d):
    """Step by step with the window of taps as a user would carry it."""
    window = [d["state"][:, i] for i in range(case["taps"] - 1)]
    ys = []
    w = d["weight"]
    for t in range(case["steps"]):
        if t > 0 and d["done"] is not None:
            over = d["done"][t - 1][:, None]
            window = [v.masked_fill(over, 0) for v in window]
        x = d["x"][t]
        live = None if d["lengths"] is None else (d["lengths"] > t)[:, None]
        if live is not None:
            x = x.masked_fill(~live, 0)
        pre = d["bias"] + x * w[:, -1]
        for i, v in enumerate(window):
            pre = pre + v * w[:, i]
        y = torch.nn.functional.silu(pre) if case["act"] == "silu" else pre
        moved = window[1:] + [x]
        if live is not None:
            y = y.masked_fill(~live, 0)
            moved = [torch.where(live, m, v) for m, v in zip(moved, window)]
            # an ended row keeps the taps of its own last step: nothing behind its end clears them
            if d["done"] is not None and t > 0:
                moved = [torch.where(live, m, v) for m, v in zip(moved, before)]
        window = moved
        before = window
        ys.append(y)
    return torch.stack(ys), torch.stack(window, 1)


def _exact_scan(case, d):
    share = case["width"] // case["groups"]
    h, ys = d["state"], []
    for t in range(case["steps"]):
        start = h
        if t > 0 and d["done"] is not None:
            start = h.masked_fill(d["done"][t - 1][:, None, None], 0)
        step = torch.nn.functional.softplus(d["delta"][t] + d["delta_bias"])
        u, z = d["u"][t], d["z"][t]
        b, c = (torch.repeat_interleave(d[k][t], share, 1) for k in ("B", "C"))
        new = start * torch.exp(step.unsqueeze(-1) * d["A"]) + b * (step * u).unsqueeze(-1)
        y = (torch.einsum("rcn,rcn->rc", new, c) + d["D"] * u) * torch.nn.functional.silu(z)
        if d["lengths"] is not None:
            live = (d["lengths"] > t)[:, None]
            y = y.masked_fill(~live, 0)
            new = torch.where(live.unsqueeze(-1), new, h)
        h = new
        ys.append(y)
    return torch.stack(ys), h


def _exact_gated(d, case):
    leaves = [d[k].requires_grad_(case["train"]) for k in _leaves(case)]
    x, wg, wu, wd = leaves
    f = torch.nn.functional
    act = f.silu if case["act"] == "silu" else f.gelu
    y = f.linear(act(f.linear(x, wg)) * f.linear(x, wu), wd)
    if not case["train"]:
        return (y,)
    return y.detach(), *torch.autograd.grad(y, leaves, d["dy"])
