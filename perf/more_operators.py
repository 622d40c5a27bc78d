"""What the policy's memory and its distillation are measured on: cases, plain forms and 64-bit values.

`own` false: elementary torch operations in 32 bits, rounded once at the end.  `own` true: the package's operators
(isaac-net_b200/policy_ops.py) as a user's program calls them: causal_conv and selective_scan over rollouts of every robot
[E, R, T, C] with the envs' resets inside, their one-step forms in the control loop, and distill_loss from a teacher's
logged top logits.
"""
import importlib
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
MOST = 1 << 30                # state elements (steps x channels x states) of the largest scan


def _ops():
    return importlib.import_module("isaac-net_b200").policy_ops


# ------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # training on 16 control steps of 1024 envs x 32 robots, the rollout buffer as it was filled: step by step
        dict(name="conv train, 1024 x 32 x 16", op="conv", e=1024, r=32, t=16, d=256, k=4, dtype="bf16", act="silu",
             carry=True, resets=0.02, major="time"),
        # config 1's batch (64 envs x 16 robots) with an odd width and length, fp32, no activation
        dict(name="conv train, 64 x 16 x 37, odd", op="conv", e=64, r=16, t=37, d=257, k=3, dtype="f32", act="none",
             carry=False, resets=0.05, major="robot"),
        # one env of 16 robots in the control loop: latency
        dict(name="conv step, 16 robots", op="conv_step", e=1, r=16, d=1024, k=4, dtype="bf16", act="silu", resets=0.0),
        # every robot of config 2 in the control loop: bound by the states' bytes
        dict(name="conv step, 4096 x 32", op="conv_step", e=4096, r=32, d=512, k=4, dtype="bf16", act="silu", resets=0.01),
        # one long log of one robot replayed through a wide memory: few rows, a long axis
        dict(name="scan 1 x 4096", op="scan", e=1, r=1, t=4096, d=2048, n=16, dtype="bf16", train=False, gate=True,
             carry=True, resets=0.0, major="robot"),
        # a training step on the rollout buffer of 1024 envs x 32 robots: the largest
        dict(name="scan train, 1024 x 32 x 16", op="scan", e=1024, r=32, t=16, d=128, n=16, dtype="bf16", train=True,
             gate=True, carry=True, resets=0.02, major="time"),
        # few long episodes of odd length and width, fp32, ten states a channel, no gate
        dict(name="scan train, 3 x 1021, odd", op="scan", e=3, r=1, t=1021, d=500, n=10, dtype="f32", train=True, gate=False,
             carry=False, resets=0.01, major="robot"),
        # one env of 16 robots in the control loop: latency
        dict(name="scan step, 16 robots", op="scan_step", e=1, r=16, d=1024, n=16, dtype="bf16", gate=True, resets=0.0),
        # every robot of config 2 in the control loop: bound by the states' bytes
        dict(name="scan step, 4096 x 32", op="scan_step", e=4096, r=32, d=256, n=16, dtype="bf16", gate=True, resets=0.01),
        # message class x priority for every robot of config 2, the actions that are not allowed masked
        dict(name="distill 131072 x 33, masked", op="distill", rows=131072, v=33, k=8, dtype="f32", tau=1.0, mask=True),
        # few rows of a large vocabulary: a long axis
        dict(name="distill 64 x 131072", op="distill", rows=64, v=131072, k=64, dtype="bf16", tau=2.0, mask=False),
        # a batch of a large vocabulary of odd size
        dict(name="distill 8192 x 32001", op="distill", rows=8192, v=32001, k=50, dtype="bf16", tau=1.0, mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def _width(rng, lo, hi):
    v = _log(rng, lo, hi)
    m = rng.choice((1, 2, 8, 64))
    return max(m, v // m * m)


def _batch(rng, most):
    """Envs and robots: at most `most` sequences."""
    r = min(rng.choice((1, 3, 16, 32)), max(1, most))
    return _log(rng, 1, max(1, min(32768, most) // r)), r


def draw(rng):
    op = rng.choice(("conv", "conv_step", "scan", "scan", "scan_step", "distill"))
    dtype = rng.choice(("bf16", "f16", "f32"))
    if op == "distill":
        v = _width(rng, 2, 131072)
        rows = _log(rng, 1, max(1, min(131072, 8192 * 32001 // v // (2 if dtype == "f32" else 1))))
        return dict(op=op, rows=rows, v=v, k=min(v, rng.choice((1, 5, 8, 32, 50, 64, 200))), dtype=dtype,
                    tau=rng.choice((1.0, 0.5, 2.0, 4.0)), mask=rng.random() < 0.4)
    resets = rng.choice((0.0, 0.01, 0.2))
    if op in ("conv", "conv_step"):
        d, k = _width(rng, 16, 4096), rng.choice((2, 3, 4))
        act = rng.choice(("silu", "none"))
        most = (1 << 27) // d // (2 if dtype == "f32" else 1)
        if op == "conv_step":
            e, r = _batch(rng, min(131072, most // 2))
            return dict(op=op, e=e, r=r, d=d, k=k, dtype=dtype, act=act, resets=resets)
        t = _log(rng, 1, 4096)
        e, r = _batch(rng, most // t)
        return dict(op=op, e=e, r=r, t=min(t, most), d=d, k=k, dtype=dtype, act=act, carry=rng.random() < 0.5, resets=resets,
                    major=rng.choice(("time", "robot")))
    d, n = _width(rng, 16, 2048), rng.choice((4, 8, 16, 16, 16, 32, 64, 5, 10))
    gate = rng.random() < 0.7
    most = MOST // (d * n)
    if op == "scan_step":
        e, r = _batch(rng, min(131072, most // 2))
        return dict(op=op, e=e, r=r, d=d, n=n, dtype=dtype, gate=gate, resets=resets)
    t = _log(rng, 1, min(4096, most))
    e, r = _batch(rng, most // t // (2 if dtype == "f32" else 1))
    return dict(op=op, e=e, r=r, t=t, d=d, n=n, dtype=dtype, train=rng.random() < 0.6, gate=gate, carry=rng.random() < 0.5,
                resets=resets, major=rng.choice(("time", "robot")))


# ------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dt = dict(case), TYPES[case["dtype"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    s = dict(case=c)
    if c["op"] == "distill":
        rows, v, k = c["rows"], c["v"], c["k"]
        logits = rn(rows, v).mul_(2)
        near = torch.topk(logits + rn(rows, v), k)                       # a teacher who agrees by and large
        s["logits"] = logits.to(dt).requires_grad_(True)
        s["teacher"], s["index"] = near.values.to(dt), near.indices
        s["index"][torch.rand(rows, k, generator=gen, device=DEV) < 0.05] = -1      # a logged list that is not full
        s["g"] = torch.rand(rows, generator=gen, device=DEV) / rows
        s["mask"] = None
        if c["mask"]:
            m = torch.rand(rows, v, generator=gen, device=DEV) < 0.8
            s["mask"] = m & (torch.rand(rows, 1, generator=gen, device=DEV) >= 0.01)      # some rows allow nothing
        return s
    e, r, d = c["e"], c["r"], c["d"]
    step = c["op"].endswith("_step")
    t = 1 if step else c["t"]

    def seq(*last):
        """[E, R, T, ...] as the rollout buffer holds it: filled step by step, or one robot's steps together."""
        if step:
            return rn(e, r, *last).to(dt)
        if c["major"] == "time":
            return rn(t, e, r, *last).to(dt).permute(1, 2, 0, *range(3, 3 + len(last)))
        return rn(e, r, t, *last).to(dt)

    def fresh(*lead):
        """Which steps start an episode: one flag for the robots of an env."""
        return (torch.rand(*lead, generator=gen, device=DEV) < c["resets"]) if c["resets"] else None

    s["x"] = seq(d)
    if step:
        s["reset"] = fresh(e, 1)
    elif c["major"] == "time":
        s["reset"] = None if not c["resets"] else fresh(t, e).t()[:, None]
    else:
        s["reset"] = fresh(e, 1, t)
    if c["op"].startswith("conv"):
        s["weight"], s["bias"] = (rn(d, c["k"]) * c["k"] ** -0.5).to(dt), (rn(d) * 0.1).to(dt)
        s["state"] = rn(e, r, c["k"] - 1, d).to(dt) if step or c["carry"] else None
        names = ("x", "weight", "bias", "state")
    else:
        n = c["n"]
        bc = seq(2 * n)                                  # both from one projection
        s["b"], s["c"] = bc[..., :n], bc[..., n:]
        s["dt"] = seq(d) * 0.5
        rate = torch.exp(torch.rand(d, generator=gen, device=DEV) * math.log(100.0)) * 1e-3      # steps of 0.001 to 0.1
        s["dt_bias"] = torch.log(torch.expm1(rate))
        s["a"] = -torch.arange(1, n + 1, device=DEV) * torch.exp(0.1 * rn(d, n))
        s["d"] = 1 + 0.1 * rn(d)
        s["z"] = seq(d) if c["gate"] else None
        s["state"] = rn(e, r, d, n) if step or c["carry"] else None
        names = ("x", "dt", "a", "b", "c", "d", "z", "dt_bias", "state")
    if not step and c.get("train", True):
        s["gy"] = seq(d)
        s["wrt"] = [k for k in names if s[k] is not None]
        for k in s["wrt"]:
            s[k] = s[k].detach().requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _flat(v, last=1):
    """[E, R, T, ...] in 32 bits as [sequences, T, ...]."""
    v = v.detach().float()
    return v.reshape(-1, *v.shape[-1 - last:])


def _since(reset, e, r, t, start):
    """[sequences, T]: steps since the episode's first one; before any reset, counted from `start` steps before the call."""
    at = torch.arange(t, device=DEV)
    if reset is None:
        return (at + start).expand(e * r, t)
    first = torch.where(reset.reshape(e, t), at, -start).cummax(-1).values
    return (at - first).repeat_interleave(r, 0)


def _silu(v):
    """silu and its derivative."""
    s = 1 / (1 + torch.exp(-v))
    return v * s, s * (1 + v * (1 - s))


def _conv(s):
    c, dt = s["case"], s["x"].dtype
    e, r, t, d, k = c["e"], c["r"], c["t"], c["d"], c["k"]
    x, w, bias = _flat(s["x"]), s["weight"].detach().float(), s["bias"].detach().float()
    old = s["state"].detach().float().reshape(-1, k - 1, d) if s["state"] is not None else x.new_zeros(e * r, k - 1, d)
    xp = torch.cat((old, x), 1)
    since = _since(s["reset"], e, r, t, k - 1)
    taps = [(since >= j)[..., None] * xp[:, k - 1 - j:k - 1 - j + t] for j in range(k)]      # x_(t - j)
    pre = sum(taps[j] * w[:, k - 1 - j] for j in range(k)) + bias
    act, slope = _silu(pre) if c["act"] == "silu" else (pre, torch.ones((), device=DEV))
    last = since[:, -1:] >= torch.arange(k - 2, -1, -1, device=DEV)
    new = torch.where(last[..., None], xp[:, t:], 0)
    g = _flat(s["gy"]) * slope
    gw = torch.stack([(g * taps[k - 1 - i]).sum((0, 1)) for i in range(k)], -1)
    pad = torch.nn.functional.pad
    gxp = sum(pad((since >= j)[..., None] * g * w[:, k - 1 - j], (0, 0, k - 1 - j, j)) for j in range(k))
    outs = [act.view(e, r, t, d), new.view(e, r, k - 1, d), gxp[:, k - 1:].reshape(e, r, t, d), gw, g.sum((0, 1))]
    if s["state"] is not None:
        outs.append(gxp[:, :k - 1].reshape(e, r, k - 1, d))
    return [o.to(dt) for o in outs]


def _conv_step(s):
    c, dt = s["case"], s["x"].dtype
    x, old = s["x"].float(), s["state"].float()
    if s["reset"] is not None:
        old = torch.where(s["reset"][..., None, None], 0, old)
    win = torch.cat((old, x[..., None, :]), -2)
    pre = (win * s["weight"].float().T).sum(-2) + s["bias"].float()
    s["state"].copy_(win[..., 1:, :])
    return [(_silu(pre)[0] if c["act"] == "silu" else pre).to(dt), s["state"]]


def _softplus(v):
    return torch.log1p(torch.exp(-v.abs())) + v.clamp(min=0)


def _linear(a, b):
    """h_t = a_t h_(t-1) + b_t along axis 1, by doubling."""
    k = 1
    while k < a.shape[1]:
        b = torch.cat((b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]), 1)
        a = torch.cat((a[:, :k], a[:, k:] * a[:, :-k]), 1)
        k *= 2
    return b


def _scan(s):
    c, dt = s["case"], s["x"].dtype
    e, r, t, d, n = c["e"], c["r"], c["t"], c["d"], c["n"]
    x, raw, b, cc = (_flat(s[k]) for k in ("x", "dt", "b", "c"))
    a, dd, bias = (s[k].detach() for k in ("a", "d", "dt_bias"))
    v = raw + bias
    delta = _softplus(v)
    decay = torch.exp(delta[..., None] * a)                                   # [S, T, D, N]
    if s["reset"] is not None:
        decay = decay * (_since(s["reset"], e, r, t, t + 1) > 0)[..., None, None]
    inp = (delta * x)[..., None] * b[:, :, None]
    h0 = s["state"].detach().reshape(-1, 1, d, n) if s["state"] is not None else x.new_zeros(e * r, 1, d, n)
    inp[:, :1] += decay[:, :1] * h0
    h = _linear(decay, inp)
    del inp
    y0 = torch.einsum("stdn,stn->std", h, cc) + dd * x
    out = lambda o: o.reshape(e, r, t, -1).to(dt)
    if s["z"] is not None:
        gate, slope = _silu(_flat(s["z"]))
    y = y0 * gate if s["z"] is not None else y0
    outs = [out(y), h[:, -1].clone().view(e, r, d, n)]
    if not c["train"]:
        return outs
    gy = _flat(s["gy"])
    g = gy * gate if s["z"] is not None else gy
    later = torch.cat((decay[:, 1:], decay.new_zeros(e * r, 1, d, n)), 1)
    dh = _linear(later.flip(1), (g[..., None] * cc[:, :, None]).flip(1)).flip(1)
    del later
    before = torch.cat((h0, h[:, :-1]), 1)
    q = dh * before * decay
    s1 = torch.einsum("stdn,stn->std", dh, b)
    ddelta = torch.einsum("stdn,dn->std", q, a) + s1 * x
    graw = ddelta / (1 + torch.exp(-v))
    grads = dict(x=out(s1 * delta + dd * g), dt=out(graw), a=torch.einsum("stdn,std->dn", q, delta),
                 b=out(torch.einsum("stdn,std->stn", dh, delta * x)), c=out(torch.einsum("stdn,std->stn", h, g)),
                 d=(g * x).sum((0, 1)), dt_bias=graw.sum((0, 1)), state=(dh[:, 0] * decay[:, 0]).view(e, r, d, n))
    if s["z"] is not None:
        grads["z"] = out(gy * y0 * slope)
    return outs + [grads[k] for k in s["wrt"]]


def _scan_step(s):
    dt, x = s["x"].dtype, s["x"].float()
    delta = _softplus(s["dt"].float() + s["dt_bias"])[..., None]
    old = s["state"]
    if s["reset"] is not None:
        old = torch.where(s["reset"][..., None, None], 0, old)
    h = torch.exp(delta * s["a"]) * old + delta * x[..., None] * s["b"].float()[..., None, :]
    y = (h * s["c"].float()[..., None, :]).sum(-1) + s["d"] * x
    if s["z"] is not None:
        y = y * _silu(s["z"].float())[0]
    s["state"].copy_(h)
    return [y.to(dt), s["state"]]


def _distill(s):
    c, logits = s["case"], s["logits"].detach()
    tau = c["tau"]
    rows, v = logits.shape
    z = logits.float() / tau
    on = s["index"] >= 0
    at = s["index"].clamp(min=0)
    if s["mask"] is not None:
        z = torch.where(s["mask"], z, -math.inf)
        on = on & torch.gather(s["mask"], 1, at)
    live = on.any(-1, keepdim=True)
    m = z.max(-1, keepdim=True).values
    w = torch.exp(z - torch.where(m == -math.inf, 0, m))
    total = w.sum(-1, keepdim=True)
    tt = torch.where(on, s["teacher"].float() / tau, -math.inf)
    tt = tt - torch.where(live, tt.max(-1, keepdim=True).values, 0)
    p = torch.exp(tt)
    mass = torch.where(live, p.sum(-1, keepdim=True), 1)
    logq = torch.gather(z, 1, at) - m - torch.log(total)
    loss = torch.where(on, p / mass * (tt - torch.log(mass) - logq), 0).sum(-1) * tau * tau
    p = p / mass
    grad = torch.where(live, w / total, 0).scatter_add_(1, at, -p)
    return [loss, (grad * (s["g"] * tau)[:, None]).to(logits.dtype)]


# ------------------------------------------------------------------------------------------------------- a pass
def run(s):
    c = s["case"]
    if not own:
        return {"conv": _conv, "conv_step": _conv_step, "scan": _scan, "scan_step": _scan_step, "distill": _distill}[c["op"]](s)
    ops = _ops()
    if c["op"] == "distill":
        loss = ops.distill_loss(s["logits"], s["teacher"], s["index"], temperature=c["tau"], mask=s["mask"])
        return [loss.detach(), *torch.autograd.grad(loss, s["logits"], s["g"])]
    if c["op"].startswith("conv"):
        act = c["act"] if c["act"] != "none" else None
        if c["op"] == "conv_step":
            return [ops.causal_conv_step(s["x"], s["weight"], s["state"], s["bias"], reset=s["reset"], act=act), s["state"]]
        y, new = ops.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], reset=s["reset"], act=act)
    else:
        more = dict(d=s["d"], z=s["z"], dt_bias=s["dt_bias"], reset=s["reset"])
        args = (s["x"], s["dt"], s["a"], s["b"], s["c"])
        if c["op"] == "scan_step":
            return [ops.selective_scan_step(*args, s["state"], **more), s["state"]]
        y, new = ops.selective_scan(*args, state=s["state"], **more)
        if not c["train"]:
            return [y, new]
    return [y.detach(), new.detach(), *torch.autograd.grad(y, [s[k] for k in s["wrt"]], s["gy"])]


# ------------------------------------------------------------------------------------------------------- work
def work(case):
    c, b = case, BYTES[case["dtype"]]
    if c["op"] == "distill":
        m, k = c["rows"] * c["v"], c["rows"] * c["k"]
        return {"bytes": 2 * b * m + (m if c["mask"] else 0) + (b + 8) * k + 8 * c["rows"], "flops": 6 * m}
    rows = c["e"] * c["r"]
    flags = c["e"] * c.get("t", 1) if c["resets"] else 0
    if c["op"] == "conv_step":
        return {"bytes": 2 * b * rows * c["d"] * c["k"] + b * c["d"] * (c["k"] + 1) + flags, "flops": 2 * rows * c["d"] * c["k"]}
    if c["op"] == "conv":
        m, st = rows * c["t"] * c["d"], rows * (c["k"] - 1) * c["d"]
        return {"bytes": b * (4 * m + (3 if c["carry"] else 1) * st + 2 * c["d"] * (c["k"] + 1)) + flags, "flops": 6 * m * c["k"]}
    d, n = c["d"], c["n"]
    params = 4 * d * (n + 2)
    if c["op"] == "scan_step":
        return {"bytes": rows * (b * ((4 if c["gate"] else 3) * d + 2 * n) + 8 * d * n) + params + flags,
                "flops": rows * d * (7 * n + 20)}
    m, st = rows * c["t"], 4 * rows * d * n
    streams, flops = (4 if c["gate"] else 3), 7
    if c["train"]:
        streams, flops = streams + (4 if c["gate"] else 3), 30      # gy, and the gradients of x, dt and z
    bcs, states = (4, 3) if c["train"] else (2, 2)
    return {"bytes": b * m * (streams * d + bcs * n) + (states if c["carry"] else 1) * st
            + params * (2 if c["train"] else 1) + flags, "flops": m * d * (flops * n + 20)}


# ------------------------------------------------------------------------------------------------------- 64 bits
def _exact_rollout(s, part):
    """The values of some envs' rollouts by the recurrence itself, and by autograd their gradients."""
    c = s["case"]
    step, conv = c["op"].endswith("_step"), c["op"].startswith("conv")
    shared = ("weight", "bias") if conv else ("a", "d", "dt_bias")
    cut = lambda k, v: v if k in shared else v[part]
    leaf = {k: cut(k, v).detach().double() for k, v in s.items() if torch.is_tensor(v) and k not in ("reset", "gy")}
    if not step:
        for k in s.get("wrt", ()):
            leaf[k].requires_grad_(True)
    x = leaf["x"][:, :, None] if step else leaf["x"]
    e, r, t, d = x.shape
    reset = s["reset"]
    if reset is not None:
        reset = (reset[..., None] if step else reset)[part].expand(e, r, t)
    at = lambda k, i: leaf[k] if step else leaf[k][:, :, i]
    ys = []
    if conv:
        w, k = leaf["weight"], c["k"]
        h = leaf["state"] if leaf.get("state") is not None else x.new_zeros(e, r, k - 1, d)
        for i in range(t):
            if reset is not None:
                h = h.masked_fill(reset[:, :, i, None, None], 0.0)
            h = torch.cat((h, x[:, :, i:i + 1]), 2)
            pre = torch.einsum("erkd,dk->erd", h, w) + leaf["bias"]
            ys.append(pre * torch.sigmoid(pre) if c["act"] == "silu" else pre)
            h = h[:, :, 1:]
    else:
        h = leaf["state"] if leaf.get("state") is not None else x.new_zeros(e, r, d, c["n"])
        for i in range(t):
            if reset is not None:
                h = h.masked_fill(reset[:, :, i, None, None], 0.0)
            delta = torch.logaddexp(at("dt", i) + leaf["dt_bias"], torch.zeros((), dtype=torch.float64, device=DEV))
            h = h * torch.exp(delta[..., None] * leaf["a"]) + (delta * x[:, :, i])[..., None] * at("b", i)[:, :, None]
            y = torch.matmul(h, at("c", i)[..., None])[..., 0] + leaf["d"] * x[:, :, i]
            if leaf.get("z") is not None:
                z = at("z", i)
                y = y * z * torch.sigmoid(z)
            ys.append(y)
    y = ys[0] if step else torch.stack(ys, 2)
    outs = [y.detach(), h.detach()]
    if "gy" in s:
        outs += torch.autograd.grad(y, [leaf[k] for k in s["wrt"]], s["gy"][part].double())
    return outs


def _exact_distill(s):
    c = s["case"]
    logits = s["logits"].detach().double().requires_grad_(True)
    on, at = s["index"] >= 0, s["index"].clamp(min=0)
    z = logits / c["tau"]
    if s["mask"] is not None:
        on = on & torch.gather(s["mask"], 1, at)
        z = z.masked_fill(~s["mask"], -1e300)
    live = on.any(-1)
    logq = torch.gather(torch.log_softmax(z, -1), 1, at)
    teacher = (s["teacher"].double() / c["tau"]).masked_fill(~on, -1e300)
    logp = torch.log_softmax(teacher, -1)
    each = torch.where(on, torch.exp(logp) * (logp - logq), 0.0)
    loss = torch.where(live, each.sum(-1), 0.0) * c["tau"] ** 2
    return [loss.detach(), *torch.autograd.grad(loss, logits, s["g"].double())]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "distill":
        return _exact_distill(s)
    e = case["e"]
    each = case["r"] * case["d"] * case.get("t", 1) * case.get("n", case.get("k"))
    envs = max(1, min(e, MOST // 4 // each))
    with torch.set_grad_enabled("gy" in s):
        parts = [_exact_rollout(s, slice(i, i + envs)) for i in range(0, e, envs)]
    names = ["y", "new", *s.get("wrt", ())]
    shared = ("weight", "bias", "a", "d", "dt_bias")
    return [sum(p[i] for p in parts) if k in shared else torch.cat([p[i] for p in parts]) for i, k in enumerate(names)]
