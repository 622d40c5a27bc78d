"""What the policy operators (isaac-net_b200/policy_ops.py) are measured on: their cases, plain forms and work.

`own` false: elementary torch operations in 32 bits, rounded once at the end.  `own` true: the package's operators, as a
user's program calls them.  The operators make one residual block of a policy over NetModule's observations and its
answer: block_norm (pre-norm, post-norm, gate, residual scale), gated_ffn, counter_dropout, sample_logits.
"""
import importlib
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
M32 = 0xFFFFFFFF
CH_DROPOUT = 0x44
ONE = float(2 ** 40)          # sample_logits' fixed point


def _ops():
    return importlib.import_module("isaac-net_b200").policy_ops


# ------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one robot's decision: the smallest serving call of a wide policy
        dict(name="ffn 1 row", op="ffn", n=1, d=1024, f=2816, dtype="bf16", act="silu", train=False),
        # one env of 16 robots through a large policy: bound by the weights' bytes
        dict(name="ffn 16 rows, large", op="ffn", n=16, d=4096, f=11264, dtype="bf16", act="silu", train=False),
        # a training step on a ragged batch whose rows are not 16-byte aligned
        dict(name="ffn train, ragged", op="ffn", n=999, d=1004, f=2681, dtype="f16", act="gelu", train=True),
        # a training step on one control step of 4096 envs x 32 robots (benchmark config 2), a small policy
        dict(name="ffn train, 4096 x 32", op="ffn", n=131072, d=512, f=1408, dtype="bf16", act="silu", train=True),
        # the largest: a training step of a large policy
        dict(name="ffn train, large", op="ffn", n=8192, d=4096, f=11264, dtype="bf16", act="silu", train=True),
        # serving one env of 32 robots: the residual join of one block and the pre-norm of the next
        dict(name="norm 32 rows", op="norm", n=32, group=32, d=1024, dtype="bf16", train=False, post=True, scale=0.5),
        # training, 4096 envs x 32 robots, one gate per env (a condition shared by its robots)
        dict(name="norm train, 4096 x 32", op="norm", n=131072, group=32, d=512, dtype="bf16", train=True, post=True,
             scale=0.5),
        # training the widest hidden activations of the same batch
        dict(name="dropout, 4096 x 32", op="dropout", e=4096, r=32, d=1408, dtype="bf16", p=0.1),
        # config 1's batch (64 envs x 16 robots) with an odd width, in fp32
        dict(name="dropout, 64 x 16, odd", op="dropout", e=64, r=16, d=257, dtype="f32", p=0.5),
        # message class x priority for every robot of config 2, with the actions that are not allowed masked
        dict(name="sample 131072 x 33, masked", op="sample", n=131072, v=33, dtype="f32", temp=1.0, top_k=0, top_p=0.95,
             min_p=0.0, mask=True),
        # one row of a large vocabulary: latency
        dict(name="sample 1 x 32001", op="sample", n=1, v=32001, dtype="f32", temp=0.7, top_k=40, top_p=1.0,
             min_p=0.05, mask=False),
        # a batch of a large vocabulary with every filter on
        dict(name="sample 64 x 131072", op="sample", n=64, v=131072, dtype="bf16", temp=0.8, top_k=1000, top_p=0.9,
             min_p=0.01, mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    v = _log(rng, lo, hi)
    m = rng.choice((1, 2, 8, 64))
    return max(m, v // m * m)


def draw(rng):
    op = rng.choice(("ffn", "norm", "dropout", "sample"))
    if op == "ffn":
        d, f = _width(rng, 64, 4096), _width(rng, 64, 11264)
        train = rng.random() < 0.5
        most = 8192 * 4096 * 11264 // (d * f)
        n = _log(rng, 1, min(131072, most) if train else min(4096, most))
        return dict(op="ffn", n=n, d=d, f=f, dtype=rng.choice(("bf16", "f16")), act=rng.choice(("silu", "gelu")),
                    train=train)
    if op == "norm":
        d = _width(rng, 16, 8192)
        n = _log(rng, 1, min(131072, 131072 * 512 // d))
        group = rng.choice((0, 1, 16, 32, n))      # 0: no gate; 1: a gate per row; n: one gate for every row
        if group > 1:
            n = max(1, n // group) * group
        return dict(op="norm", n=n, group=group, d=d, dtype=rng.choice(("bf16", "f16", "f32")),
                    train=rng.random() < 0.6, post=rng.random() < 0.7, scale=rng.choice((1.0, 0.5, 0.1)))
    if op == "dropout":
        d, r = _width(rng, 16, 4096), rng.choice((1, 3, 16, 32, 100, 128))
        e = _log(rng, 1, max(1, min(8192, 131072 * 1408 // (r * d))))
        return dict(op="dropout", e=e, r=r, d=d, dtype=rng.choice(("bf16", "f16", "f32")),
                    p=rng.choice((0.0, 0.1, 0.25, 0.5, 0.9)))
    v = _width(rng, 2, 131072)
    n = _log(rng, 1, max(1, min(131072, 64 * 131072 // v)))
    return dict(op="sample", n=n, v=v, dtype=rng.choice(("bf16", "f16", "f32")), temp=rng.choice((0.0, 0.6, 1.0, 1.5)),
                top_k=rng.choice((0, 0, 1, 8, 50, 1000)), top_p=rng.choice((1.0, 0.95, 0.6)),
                min_p=rng.choice((0.0, 0.05, 0.2)), mask=rng.random() < 0.4)


# ------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dt = dict(case), TYPES[case["dtype"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    s = dict(case=c)
    if c["op"] == "ffn":
        n, d, f = c["n"], c["d"], c["f"]
        s["x"] = rn(n, d).to(dt)                                    # normalised activations
        s["wg"], s["wu"] = ((rn(f, d) * d ** -0.5).to(dt) for _ in range(2))
        s["wd"] = (rn(d, f) * f ** -0.5).to(dt)
        if c["train"]:
            s["dy"] = rn(n, d).to(dt)
            for k in ("x", "wg", "wu", "wd"):
                s[k].requires_grad_(True)
    elif c["op"] == "norm":
        n, d = c["n"], c["d"]
        s["x"], s["h"] = (rn(n, d) * 2).to(dt), (rn(n, d) * 0.7).to(dt)
        s["win"] = (1 + 0.1 * rn(d)).to(dt)
        s["wpost"] = (1 + 0.1 * rn(d)).to(dt) if c["post"] else None
        if c["group"]:
            s["gate"] = (0.5 + 0.5 * rn(n // c["group"], d)).to(dt)
        else:
            s["gate"] = None
        if c["train"]:
            s["gy"], s["gn"] = rn(n, d).to(dt), rn(n, d).to(dt)
            for k in ("x", "h", "win", "wpost", "gate"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    elif c["op"] == "dropout":
        e = c["e"]
        s["x"] = rn(e, c["r"], c["d"]).to(dt).requires_grad_(True)
        s["gy"] = rn(e, c["r"], c["d"]).to(dt)
        s["s0"] = (seed * 2654435761 + 12345) & M32
        s["env"] = torch.arange(e, device=DEV) + 1000
        s["episode"] = torch.randint(0, 50, (e,), generator=gen, device=DEV)
        s["ctr"] = torch.randint(0, 1000, (e,), generator=gen, device=DEV)
    else:
        n, v = c["n"], c["v"]
        s["logits"] = (rn(n, v) * 3).to(dt)
        s["u"] = torch.rand(n, generator=gen, device=DEV)
        s["mask"] = None
        if c["mask"]:
            m = torch.rand(n, v, generator=gen, device=DEV) < 0.7
            m &= torch.rand(n, 1, generator=gen, device=DEV) >= 0.01    # some rows allow nothing
            s["mask"] = m
    return s


# ------------------------------------------------------------------------------------------------------- plain forms
def _act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        t = 1 / (1 + torch.exp(-g))
        return g * t, t * (1 + g * (1 - t))
    c = 0.5 * (1 + torch.erf(g * 0.7071067811865476))
    return g * c, c + g * torch.exp(-0.5 * g * g) * 0.3989422804014327


def _ffn(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[k].detach().float() for k in ("x", "wg", "wu", "wd"))
    g, u = x @ wg.T, x @ wu.T
    a, da = _act(g, c["act"])
    h = a * u
    y = (h @ wd.T).to(dt)
    if not c["train"]:
        return y
    dy = s["dy"].float()
    dh = dy @ wd
    dg, du = dh * u * da, dh * a
    return [t.to(dt) for t in (y, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ h)]


def _norm(s):
    c, dt = s["case"], s["x"].dtype
    f = lambda t: None if t is None else t.detach().float()
    x, h, win, wpost, gate = f(s["x"]), f(s["h"]), f(s["win"]), f(s["wpost"]), f(s["gate"])
    n, d, sc = c["n"], c["d"], c["scale"]
    g = gate.repeat_interleave(c["group"], 0) if gate is not None else torch.ones((), device=x.device)
    rh = (h.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hh = h * rh
    p = hh * wpost if wpost is not None else h
    y = x + sc * g * p
    ry = (y.square().mean(-1, keepdim=True) + EPS).rsqrt()
    yh = y * ry
    outs = [y.to(dt), (yh * win).to(dt)]
    if not c["train"]:
        return outs
    gy, gn = s["gy"].float(), s["gn"].float()
    q = gn * win
    t = gy + ry * (q - yh * (q * yh).mean(-1, keepdim=True))
    outs.append(t.to(dt))
    gp = sc * g * t
    if wpost is not None:
        q = gp * wpost
        outs.append((rh * (q - hh * (q * hh).mean(-1, keepdim=True))).to(dt))
    else:
        outs.append(gp.to(dt))
    outs.append((gn * yh).sum(0).to(dt))
    if wpost is not None:
        outs.append((gp * hh).sum(0).to(dt))
    if gate is not None:
        outs.append((sc * t * p).view(-1, c["group"], d).sum(1).to(dt))
    return outs


def _mix(v):
    v = v ^ (v >> 16)
    v = (v * 0x21F0AAAD) & M32
    v = v ^ (v >> 15)
    v = (v * 0x735A2D97) & M32
    return v ^ (v >> 15)


def _salt(v):
    return (_mix(v & M32) + 0x9E3779B9) & M32


def _dropout(s):
    c, x, gy = s["case"], s["x"].detach(), s["gy"]
    h = torch.full_like(s["env"], s["s0"])
    for word in (s["env"], s["episode"], torch.full_like(s["env"], CH_DROPOUT), s["ctr"], torch.full_like(s["env"], 3)):
        h = _mix(h ^ _salt(word))
    n = c["r"] * c["d"]
    j = torch.arange((n + 1) // 2, device=x.device)
    base = h[:, None]
    w = _mix(_mix((base + j * 0x9E3779B9) & M32) ^ base)
    t = round(c["p"] * 65536)
    keep = (torch.stack((w & 0xFFFF, w >> 16), -1).view(c["e"], -1)[:, :n] >= t).view(x.shape)
    scale = 65536 / (65536 - t) if t < 65536 else 0.0
    zero = torch.zeros((), device=x.device)
    return [torch.where(keep, v.float() * scale, zero).to(x.dtype) for v in (x, gy)]


def _sample(s):
    c, l, u = s["case"], s["logits"].float(), s["u"]
    n, v = l.shape
    l = torch.where(torch.isnan(l), -math.inf, l)
    if s["mask"] is not None:
        l = torch.where(s["mask"], l, -math.inf)
    m = l.max(-1, keepdim=True).values
    dead = m == -math.inf
    z = torch.where(l == m, 0.0, (l - m) * (1 / np.float32(c["temp"]) if c["temp"] > 0 else np.float32(1)).item())
    w = torch.where(dead, 0.0, torch.exp(z))
    q = (w.double() * ONE).long()
    k = 1 if c["temp"] == 0 else c["top_k"]
    if k > 0 or c["top_p"] < 1:
        order = torch.sort(l, dim=-1, descending=True, stable=True).indices
        qs = torch.gather(q, 1, order)
        if 0 < k < v:
            qs[:, k:] = 0
        keep = torch.arange(v, device=l.device)[None] < (k if k > 0 else v)
        if c["top_p"] < 1:
            before = qs.cumsum(-1) - qs
            keep = keep & (before.double() < float(np.float32(c["top_p"])) * qs.sum(-1, keepdim=True).double())
            keep[:, 0] = True
        keep = torch.zeros_like(q, dtype=torch.bool).scatter_(1, order, keep.expand(n, v))
        q = torch.where(keep, q, 0)
    if c["min_p"] > 0:
        q = torch.where(w >= np.float32(c["min_p"]).item(), q, 0)
    run = q.cumsum(-1)
    total = run[:, -1:]
    at = (u[:, None].double() * total.double()).long().minimum(total - 1)
    token = (run > at).to(torch.uint8).argmax(-1)
    zt = torch.gather(z, 1, token[:, None]).double()
    logp = (zt - torch.log(total.double() / ONE))[:, 0]
    dead = dead[:, 0]
    return [torch.where(dead, -1, token), torch.where(dead, -math.inf, logp).float()]


# ------------------------------------------------------------------------------------------------------- a pass
def run(s):
    c = s["case"]
    if not own:
        return {"ffn": _ffn, "norm": _norm, "dropout": _dropout, "sample": _sample}[c["op"]](s)
    ops = _ops()
    if c["op"] == "ffn":
        args = (s["x"], s["wg"], s["wu"], s["wd"])
        y = ops.gated_ffn(*args, act=c["act"])
        if not c["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, args, s["dy"])]
    if c["op"] == "norm":
        x, h, gate, n, d = s["x"], s["h"], s["gate"], c["n"], c["d"]
        if gate is not None and c["group"] > 1:      # one gate for each group of rows: [groups, rows, D] with [groups, 1, D]
            x, h = x.view(-1, c["group"], d), h.view(-1, c["group"], d)
            g = gate.view(-1, 1, d)
        else:
            g = gate
        y, o = ops.block_norm(x, s["win"], h, post_weight=s["wpost"], gate=g, scale=c["scale"], eps=EPS)
        if not c["train"]:
            return [y.view(n, d), o.view(n, d)]
        wrt = [t for t in (s["x"], s["h"], s["win"], s["wpost"], gate) if t is not None]
        grads = torch.autograd.grad((y, o), wrt, (s["gy"].view(y.shape), s["gn"].view(y.shape)))
        return [y.detach().view(n, d), o.detach().view(n, d), *grads]
    if c["op"] == "dropout":
        y = ops.counter_dropout(s["x"], c["p"], s["s0"], s["env"], s["episode"], s["ctr"], stream=3)
        return [y.detach(), *torch.autograd.grad(y, s["x"], s["gy"])]
    return list(ops.sample_logits(s["logits"], s["u"], temperature=c["temp"], top_k=c["top_k"], top_p=c["top_p"],
                                  min_p=c["min_p"], mask=s["mask"]))


# ------------------------------------------------------------------------------------------------------- work
def work(case):
    c, b = case, BYTES[case["dtype"]]
    if c["op"] == "ffn":
        n, d, f = c["n"], c["d"], c["f"]
        if not c["train"]:
            return {"bytes": b * (3 * d * f + 2 * n * d), "flops": 6 * n * d * f}
        return {"bytes": b * (6 * d * f + 4 * n * d), "flops": 18 * n * d * f}
    if c["op"] == "norm":
        n, d = c["n"], c["d"]
        gates = n // c["group"] if c["group"] else 0
        rows, vecs = (8, 2) if c["train"] else (4, 1)
        return {"bytes": b * d * (rows * n + vecs * (gates + 1 + c["post"])), "flops": (40 if c["train"] else 10) * n * d}
    if c["op"] == "dropout":
        m = c["e"] * c["r"] * c["d"]
        return {"bytes": 4 * b * m + 24 * c["e"], "flops": 2 * m}
    m = c["n"] * c["v"]
    return {"bytes": (b + (1 if c["mask"] else 0)) * m + 16 * c["n"], "flops": 4 * m}


# ------------------------------------------------------------------------------------------------------- 64 bits
def _exact_ffn(s):
    c = s["case"]
    x, wg, wu, wd = (s[k].detach().double() for k in ("x", "wg", "wu", "wd"))
    g, u = torch.einsum("nd,fd->nf", x, wg), torch.einsum("nd,fd->nf", x, wu)
    if c["act"] == "silu":
        sg = torch.sigmoid(g)
        a, da = g * sg, sg + g * sg * torch.sigmoid(-g)
    else:
        cdf = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        a, da = g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    y = torch.einsum("nf,df->nd", a * u, wd)
    if not c["train"]:
        return y
    dy = s["dy"].double()
    dh = torch.einsum("nd,df->nf", dy, wd)
    dwd = torch.einsum("nd,nf->df", dy, a * u)
    dg = dh * u * da
    dwg = torch.einsum("nf,nd->fd", dg, x)
    dx = torch.einsum("nf,fd->nd", dg, wg)
    du = dh * a
    return [y, dx + torch.einsum("nf,fd->nd", du, wu), dwg, torch.einsum("nf,nd->fd", du, x), dwd]


def _exact_norm(s):
    c = s["case"]
    leaf = {k: s[k].detach().double().requires_grad_(c["train"]) for k in ("x", "h", "win", "wpost", "gate")
            if s[k] is not None}
    rms = lambda v: v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    a = rms(leaf["h"]) * leaf["wpost"] if "wpost" in leaf else leaf["h"]
    if "gate" in leaf:
        a = (a.view(-1, c["group"], c["d"]) * leaf["gate"][:, None]).view(c["n"], c["d"])
    y = leaf["x"] + c["scale"] * a
    n = rms(y) * leaf["win"]
    if not c["train"]:
        return [y, n]
    grads = torch.autograd.grad((y, n), list(leaf.values()), (s["gy"].double(), s["gn"].double()))
    return [y.detach(), n.detach(), *grads]


def _exact_dropout(s):
    c = s["case"]
    u32 = np.uint32

    def mix(v):
        v = v ^ (v >> u32(16))
        v *= u32(0x21F0AAAD)
        v ^= v >> u32(15)
        v *= u32(0x735A2D97)
        v ^= v >> u32(15)
        return v

    e, n = c["e"], c["r"] * c["d"]
    key = np.full(e, s["s0"], u32)
    for word in (s["env"].cpu().numpy(), s["episode"].cpu().numpy(), np.full(e, CH_DROPOUT), s["ctr"].cpu().numpy(),
                 np.full(e, 3)):
        key = mix(key ^ (mix(word.astype(u32)) + u32(0x9E3779B9)))
    j = np.arange((n + 1) // 2, dtype=u32) * u32(0x9E3779B9)
    t = round(c["p"] * 65536)
    keep = np.empty((e, n), bool)
    for i in range(e):
        h = mix(mix(key[i] + j) ^ key[i])
        keep[i] = np.stack((h & u32(0xFFFF), h >> u32(16)), -1).reshape(-1)[:n] >= t
    k = torch.from_numpy(keep).to(DEV).view(s["x"].shape)
    return [(v.detach().double() / (1 - t / 65536)).masked_fill(~k, 0) for v in (s["x"], s["gy"])]


def _exact_sample(s):
    c = s["case"]
    l = s["logits"].double()
    if s["mask"] is not None:
        l = l.masked_fill(~s["mask"], -math.inf)
    dead = ~torch.isfinite(l).any(-1)
    l = torch.where(dead[:, None], 0.0, l)
    n, v = l.shape
    srt, order = torch.sort(l, dim=-1, descending=True, stable=True)
    k = 1 if c["temp"] == 0 else c["top_k"] or v
    pr = torch.softmax(srt / float(np.float32(c["temp"] or 1)), -1)
    pr[:, k:] = 0
    pr = pr / pr.sum(-1, keepdim=True)
    if c["top_p"] < 1:
        out = pr.cumsum(-1) - pr >= float(np.float32(c["top_p"]))
        out[:, 0] = False
        pr = pr.masked_fill(out, 0)
    pr = pr.masked_fill(pr < float(np.float32(c["min_p"])) * pr[:, :1], 0)
    pr = torch.zeros_like(pr).scatter_(1, order, pr / pr.sum(-1, keepdim=True))
    token = (pr.cumsum(-1) > s["u"].double()[:, None]).to(torch.uint8).argmax(-1)
    logp = torch.log(torch.gather(pr, 1, token[:, None]))[:, 0]
    return [None, torch.where(dead, -math.inf, logp)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"ffn": _exact_ffn, "norm": _exact_norm, "dropout": _exact_dropout, "sample": _exact_sample}[case["op"]](s)
