"""The policy operators block_norm, counter_dropout and sample_logits against plain 64-bit forms.

Tolerances: an output is rounded once to its type (unit roundoff U) from fp32 arithmetic.  A value made of sums of n
fp32 terms carries at most L roundings of 2^-24 of the sum of the terms' absolute values, L the longest chain of adds:
here at most 64 for a row (elements of a thread plus the tree) and 1024 for a column (rows of a worker plus the tree).
Tokens and masks are whole: they must be equal.
"""
import importlib
import math

import numpy as np
import pytest
import torch

ib = importlib.import_module("isaac-net_b200")
ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
ROW, COL = 64 * 2.0 ** -24, 1024 * 2.0 ** -24
DT = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


def near(got, ref, mag, what, dtype=None):
    """|got - ref| <= U |ref| + mag, element by element (and the smallest subnormal of the type)."""
    u = U[dtype or got.dtype]
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 1e-37
    err = (got.double() - ref).abs()
    bound = u * 1.01 * ref.abs() + mag + tiny
    assert bool((err <= bound).all()), f"{what}: worst {float((err / bound).max()):.2f} of the bound"


# ---------------------------------------------------------------------------------------------------- block_norm
def norm_ref(x, w, h, post, gate, scale, eps):
    """y, n in 64 bits; gate already of x's shape."""
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    if h is None:
        return None, rms(x) * w
    p = rms(h) * post if post is not None else h
    y = x + scale * (gate * p if gate is not None else p)
    return y, rms(y) * w


NORM = [  # leading shape, D, gate's leading shape (None: no gate), post
    ((1,), 1, None, True), ((1,), 8, (1,), True), ((3,), 7, None, False), ((5,), 33, (5,), True),
    ((4, 3), 64, (4, 1), True), ((64, 16), 257, (64, 1), True), ((2, 1000), 512, (2, 1), True),
    ((700,), 1024, (1,), False), ((37,), 1004, (37,), True), ((9,), 2050, None, True), ((6,), 4100, (1,), True),
    ((3,), 8192, (3,), True), ((3,), 8191, (1,), True), ((2500,), 256, (), True),
]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("lead,d,gl,post", NORM)
def test_block_norm_forward_and_backward(lead, d, gl, post, dtype):
    g = gen(d + len(lead))
    mk = lambda *s, a=1.0, b=0.0: (b + a * rn(g, *s)).to(dtype).requires_grad_(True)
    x, h, w = mk(*lead, d, a=2.0), mk(*lead, d, a=0.5), mk(d, a=0.2, b=1.0)
    wp = mk(d, a=0.2, b=1.0) if post else None
    gate = mk(*gl, d, a=0.5, b=0.5) if gl is not None else None
    scale, eps = 0.7, 1e-5
    y, n = ops.block_norm(x, w, h, post_weight=wp, gate=gate, scale=scale, eps=eps)
    gy, gn = rn(g, *lead, d).to(dtype), rn(g, *lead, d).to(dtype)
    args = [t for t in (x, h, w, wp, gate) if t is not None]
    grads = torch.autograd.grad((y, n), args, (gy, gn))
    # 64 bits, by autograd of the formula
    lf = [t.detach().double().requires_grad_(True) for t in args]
    it = iter(lf)
    x6, h6, w6 = next(it), next(it), next(it)
    p6 = next(it) if post else None
    g6 = next(it) if gate is not None else None
    y6, n6 = norm_ref(x6, w6, h6, p6, g6, float(np.float32(scale)), float(np.float32(eps)))
    ref = torch.autograd.grad((y6, n6), lf, (gy.double(), gn.double()))
    big = lambda t: t.abs().amax(-1, keepdim=True)
    near(y, y6.detach(), ROW * big(y6.detach()), "y")
    near(n, n6.detach(), ROW * big(n6.detach()), "n")
    near(grads[0], ref[0], 4 * ROW * big(ref[0]), "grad x")
    near(grads[1], ref[1], 4 * ROW * (big(ref[1]) + big(ref[0])), "grad h")
    yh = (y6 * (y6.square().mean(-1, keepdim=True) + 1e-5).rsqrt()).detach().abs().view(-1, d)
    near(grads[2], ref[2], COL * (gn.double().abs().view(-1, d) * yh).sum(0), "grad weight")
    if post:
        hh = (h6 * (h6.square().mean(-1, keepdim=True) + 1e-5).rsqrt()).detach().abs().view(-1, d)
        gp = ref[0].abs().view(-1, d) * scale
        if gate is not None:
            gp = gp * gate.detach().double().abs().expand(*lead, d).reshape(-1, d)
        near(grads[3], ref[3], COL * (gp * hh).sum(0), "grad post_weight")
    if gate is not None:
        p = (torch.ones_like(h6) if p6 is None else p6.detach()) * (
            h6 if p6 is None else h6 * (h6.square().mean(-1, keepdim=True) + 1e-5).rsqrt()).detach()
        terms = (ref[0] * p * scale).abs()
        mag = terms.sum_to_size(gate.shape) if gate.shape != terms.shape else terms
        # the terms are products with t = grad x, which carries the error that "grad x" above is held to
        moved = (4 * ROW * big(ref[0]) * p.abs() * scale).expand(terms.shape)
        moved = moved.sum_to_size(gate.shape) if gate.shape != terms.shape else moved
        near(grads[-1], ref[-1], COL * mag + moved, "grad gate")
    # without autograd the same values; equal inputs give equal bits
    with torch.no_grad():
        y2, n2 = ops.block_norm(x, w, h, post_weight=wp, gate=gate, scale=scale, eps=eps)
    assert torch.equal(y, y2) and torch.equal(n, n2)
    y3, n3 = ops.block_norm(x, w, h, post_weight=wp, gate=gate, scale=scale, eps=eps)
    for a, b in zip(grads, torch.autograd.grad((y3, n3), args, (gy, gn))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DT)
def test_block_norm_pre_norm_alone_and_single_outputs(dtype):
    g = gen(1)
    x, w = rn(g, 21, 96).to(dtype).requires_grad_(True), rn(g, 96).to(dtype).requires_grad_(True)
    h = rn(g, 21, 96).to(dtype).requires_grad_(True)
    n = ops.block_norm(x, w)
    gn = rn(g, 21, 96).to(dtype)
    gx, gw = torch.autograd.grad(n, (x, w), gn)
    x6, w6 = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
    n6 = norm_ref(x6, w6, None, None, None, 1.0, 1e-6)[1]
    rx, rw = torch.autograd.grad(n6, (x6, w6), gn.double())
    near(n, n6.detach(), ROW * n6.abs().max().item(), "n")
    near(gx, rx, 4 * ROW * rx.abs().max().item(), "grad x")
    near(gw, rw, COL * 21 * 4, "grad w")
    # only y used: the gradient of n is zero, that of weight too
    y, _ = ops.block_norm(x, w, h, scale=0.5)
    gx, gw, gh = torch.autograd.grad(y, (x, w, h), gn, allow_unused=True)
    assert torch.equal(gx, gn) and not bool(gw.any())
    near(gh, 0.5 * gn.double(), 0.0, "grad h")


def test_block_norm_strides_rows_and_expanded_gradients():
    g = gen(2)
    wide = rn(g, 40, 200).bfloat16()
    x, h = wide[:, 8:72], wide[:, 101:165]                 # 16-byte aligned rows, and rows that are not
    w = rn(g, 64).bfloat16()
    a = ops.block_norm(x, w, h, scale=0.3)
    b = ops.block_norm(x.contiguous(), w, h.contiguous(), scale=0.3)
    for s, t in zip(a, b):
        near(s, t.double(), ROW * t.abs().max().item(), "strided")
    xt = rn(g, 64, 40).bfloat16().t()                       # rows that are not contiguous
    near(ops.block_norm(xt, w), ops.block_norm(xt.contiguous(), w).double(), 0.0, "transposed")
    x1 = x.detach().clone().requires_grad_(True)
    n = ops.block_norm(x1, w)
    n.sum().backward()                                      # the gradient of n is one expanded element
    x2 = x.detach().clone().requires_grad_(True)
    n2 = ops.block_norm(x2, w)
    n2.backward(torch.ones_like(n2))
    assert torch.equal(x1.grad, x2.grad)


def test_block_norm_empty_zero_rows_and_gradient_differences():
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    n = ops.block_norm(x, w)
    gx, gw = torch.autograd.grad(n.sum(), (x, w))
    assert n.shape == (0, 16) and gx.shape == (0, 16) and not bool(gw.any())
    z = torch.zeros(3, 16, device="cuda")
    assert torch.equal(ops.block_norm(z, w.detach()), z)
    # directional difference of a scalar of both outputs (fp32, step 2^-7: error of order step^2 and 2^-24 / step)
    g = gen(3)
    x, h, w, p, gt = rn(g, 8, 48), rn(g, 8, 48), rn(g, 48), rn(g, 48), rn(g, 2, 1, 48)
    cy, cn = rn(g, 8, 48), rn(g, 8, 48)

    def f(s):
        t = [v + s * d for v, d in zip(base, dirs)]
        y, n = ops.block_norm(t[0].view(2, 4, 48), t[2], t[1].view(2, 4, 48), post_weight=t[3], gate=t[4], scale=0.5)
        return (y.view(8, 48).double() * cy).sum() + (n.view(8, 48).double() * cn).sum()

    base, dirs = [x, h, w, p, gt], [rn(g, *t.shape) * 0.1 for t in (x, h, w, p, gt)]
    leaf = [t.clone().requires_grad_(True) for t in base]
    y, n = ops.block_norm(leaf[0].view(2, 4, 48), leaf[2], leaf[1].view(2, 4, 48), post_weight=leaf[3], gate=leaf[4],
                          scale=0.5)
    gr = torch.autograd.grad(((y.view(8, 48) * cy).sum() + (n.view(8, 48) * cn).sum()), leaf)
    want = sum(float((a.double() * d).sum()) for a, d in zip(gr, dirs))
    step = 2.0 ** -7
    got = float(f(step) - f(-step)) / (2 * step)
    assert abs(got - want) <= 1e-3 * (abs(want) + 1.0)


# ---------------------------------------------------------------------------------------------------- counter_dropout
def drop_keys(s0, env, ep, ctr, stream):
    mix, salt = eng_mod._mix32, eng_mod._salt
    out = []
    for e, p, c in zip(env, ep, ctr):
        h = mix(s0 ^ salt(e))
        for v in (p, 0x44, c, stream):
            h = mix(h ^ salt(v))
        out.append(h)
    return out


def drop_ref(x, p, s0, env, ep, ctr, stream):
    """keep mask [E, n] and scale, word by word from the engine's own host hash."""
    e, n = x.shape[0], x[0].numel() if x.shape[0] else 0
    t = round(p * 65536)
    mix = eng_mod._mix32
    keep = torch.zeros(e, n, dtype=torch.bool)
    for i, k in enumerate(drop_keys(s0, env, ep, ctr, stream)):
        for j in range((n + 1) // 2):
            w = mix(mix((k + j * 0x9E3779B9) & 0xFFFFFFFF) ^ k)
            keep[i, 2 * j] = (w & 0xFFFF) >= t
            if 2 * j + 1 < n:
                keep[i, 2 * j + 1] = (w >> 16) >= t
    return keep.view(x.shape).cuda(), (65536 / (65536 - t) if t < 65536 else 0.0)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("shape,p", [((1, 1), 0.5), ((3, 5), 0.25), ((2, 8), 0.9), ((4, 3, 7), 0.1), ((2, 16, 260), 0.5),
                                     ((3, 4097), 0.3), ((2, 64), 0.0), ((2, 64), 1.0), ((0, 4), 0.5), ((3, 0), 0.5)])
def test_counter_dropout_equals_the_host_hash(shape, p, dtype):
    g = gen(11)
    x = rn(g, *shape).to(dtype).requires_grad_(True)
    env, ep, ctr = ([7 + 3 * i for i in range(shape[0])], [i % 2 for i in range(shape[0])],
                    [2 ** 33 + i for i in range(shape[0])])
    dev = [torch.tensor(v, dtype=torch.int64, device="cuda") for v in (env, ep, ctr)]
    s0 = eng_mod.seed_key(1234567890123)
    y = ops.counter_dropout(x, p, s0, *dev, stream=5)
    gy = rn(g, *shape).to(dtype)
    gx, = torch.autograd.grad(y, x, gy)
    if x.numel() == 0:
        assert y.shape == x.shape
        return
    keep, scale = drop_ref(x, p, s0, env, ep, ctr, 5)
    zero = torch.zeros((), device="cuda")
    assert torch.equal(y, torch.where(keep, x.detach().float() * scale, zero).to(dtype))
    assert torch.equal(gx, torch.where(keep, gy.float() * scale, zero).to(dtype))
    assert torch.equal(y, ops.counter_dropout(x.detach(), p, s0, *dev, stream=5))


def test_counter_dropout_shards_streams_and_moved_counters():
    g = gen(12)
    x = rn(g, 12, 4, 66).requires_grad_(True)
    env, ep = torch.arange(100, 112, device="cuda"), torch.zeros(12, dtype=torch.int64, device="cuda")
    ctr = torch.arange(12, device="cuda")
    full = ops.counter_dropout(x, 0.4, 99, env, ep, ctr)
    part = [ops.counter_dropout(x[i:i + 5], 0.4, 99, env[i:i + 5], ep[i:i + 5], ctr[i:i + 5]) for i in (0, 5, 10)]
    assert torch.equal(full, torch.cat(part))
    assert not torch.equal(full, ops.counter_dropout(x, 0.4, 99, env, ep, ctr, stream=1))
    assert torch.equal(ops.counter_dropout(x, 0.4, 99, env), ops.counter_dropout(x, 0.4, 99, env, ep, ep))
    mask = full != 0
    env.add_(1)
    ctr.add_(1)                                   # as the engine's next step would
    gx, = torch.autograd.grad(full, x, torch.ones_like(full))
    assert torch.equal(gx != 0, mask)
    # dropped places hold 0 whatever was there
    bad = torch.full((12, 4, 66), math.nan, device="cuda")
    out = ops.counter_dropout(bad, 0.4, 99, env - 1, ep, ctr - 1)
    assert torch.equal(torch.isnan(out), mask) and not bool(out[~mask].any())
    rate = float((ops.counter_dropout(torch.ones(64, 40000, device="cuda"), 0.3, 5, torch.arange(64, device="cuda")) == 0)
                 .double().mean())
    assert abs(rate - round(0.3 * 65536) / 65536) < 6 * math.sqrt(0.21 / (64 * 40000))


# ---------------------------------------------------------------------------------------------------- sample_logits
def sample_ref(logits, u, t, k, p, mp, mask):
    """The operator's definition row by row on the host (fp32 weights by torch on the device, the rest exact)."""
    n, v = logits.shape
    l = logits.float()
    l = torch.where(torch.isnan(l), -math.inf, l)
    if mask is not None:
        l = torch.where(mask, l, -math.inf)
    m = l.max(-1, keepdim=True).values
    it = torch.tensor([float(np.float32(1) / np.float32(a)) if a > 0 else 1.0 for a in t], device=l.device,
                      dtype=torch.float32)[:, None]
    z = torch.where(l == m, torch.zeros((), device=l.device), (l - m) * it)
    w = torch.exp(z)
    q = torch.where(l == -math.inf, torch.zeros_like(w), w).double().mul(2.0 ** 40).long()
    l, z, w, q = l.cpu(), z.cpu(), w.cpu(), q.cpu()
    tok, lp = [], []
    for r in range(n):
        if float(m[r]) == -math.inf:
            tok.append(-1)
            lp.append(-math.inf)
            continue
        order = sorted(range(v), key=lambda i: (-float(l[r, i]), i))
        kk = 1 if not t[r] > 0 else k[r]
        kept = order[:kk] if kk > 0 else order
        kept = [i for i in kept if int(q[r, i]) > 0]
        total = sum(int(q[r, i]) for i in kept)
        if p[r] < 1:
            out, before, thr = [], 0, float(np.float32(p[r])) * float(total)
            for i in kept:
                if out and float(before) >= thr:
                    break
                out.append(i)
                before += int(q[r, i])
            kept = out
        kept = sorted(i for i in kept if float(w[r, i]) >= float(np.float32(mp[r])) or float(l[r, i]) == float(m[r]))
        total = sum(int(q[r, i]) for i in kept)
        at = min(int(float(u[r]) * float(total)), total - 1)
        run = 0
        for i in kept:
            run += int(q[r, i])
            if run > at:
                break
        tok.append(i)
        lp.append(float(z[r, i]) - math.log(total / 2.0 ** 40))
    return torch.tensor(tok), torch.tensor(lp, dtype=torch.float64)


def check_sample(logits, u, t=1.0, k=0, p=1.0, mp=0.0, mask=None, rows=False):
    n = logits.shape[0]
    ls = [[a] * n if not isinstance(a, list) else a for a in (t, k, p, mp)]
    full = mask if mask is None or mask.dim() == 2 else mask.expand(logits.shape)
    want, lp = sample_ref(logits, u, *ls, full)
    if rows:
        dt = (torch.float32, torch.int32, torch.float32, torch.float32)
        t, k, p, mp = (torch.tensor(a, dtype=d, device="cuda") for a, d in zip(ls, dt))
    tok, got = ops.sample_logits(logits, u, temperature=t, top_k=k, top_p=p, min_p=mp, mask=mask)
    assert torch.equal(tok.cpu(), want), (tok.cpu() != want).nonzero().flatten()[:8]
    fin = torch.isfinite(lp)
    assert torch.equal(torch.isfinite(got.cpu()), fin)
    err = (got.cpu().double() - lp)[fin].abs()
    assert bool((err <= 2.0 ** -23 * (1 + lp[fin].abs())).all())


SIZES = [1, 2, 17, 32, 33, 64, 65, 128, 129, 255, 1000, 4096, 4097, 9001]
FILTERS = [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.1),
           (0.8, 20, 0.6, 0.02), (2.0, 1, 0.5, 0.5), (1.0, 100000, 0.999, 0.0), (1.0, 3, 0.0, 0.0)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", SIZES)
def test_sample_logits_filters(v, dtype):
    g = gen(v)
    for i, (t, k, p, mp) in enumerate(FILTERS):
        n = 6 if v > 2000 else 20
        logits = (rn(g, n, v) * 3).to(dtype)
        check_sample(logits, torch.rand(n, generator=g, device="cuda"), t, k, p, mp,
                     torch.rand(n, v, generator=g, device="cuda") < 0.5 if i % 2 else None)


@pytest.mark.parametrize("v", [3, 33, 100, 300, 5000])
def test_sample_logits_ties_infinities_and_empty_rows(v):
    g = gen(5 * v)
    u = torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24, 0.999], device="cuda")
    flat = torch.zeros(5, v, device="cuda")
    few = torch.randint(-2, 3, (5, v), generator=g, device="cuda").float()
    inf = few.clone()
    inf[:, ::3] = math.inf
    nan = few.clone()
    nan[:, ::2] = math.nan
    low = torch.full((5, v), torch.finfo(torch.float32).min, device="cuda")
    zero = few * 0.0 * torch.where(few > 0, -1.0, 1.0)       # both zeros
    dead = few.clone()
    dead[0], dead[1] = -math.inf, math.nan
    spread = few * 1e30
    for logits in (flat, few, inf, nan, low, zero, dead, spread):
        for t, k, p, mp in ((1.0, 0, 1.0, 0.0), (1.0, 2, 1.0, 0.0), (0.5, v - 1, 0.5, 0.0), (0.0, 0, 1.0, 0.0),
                            (1.0, 0, 0.3, 0.3)):
            check_sample(logits, u, t, k, p, mp)
    none = torch.zeros(5, v, dtype=torch.bool, device="cuda")
    one = none.clone()
    one[:, v // 2] = True
    check_sample(few, u, mask=none, p=0.5)
    check_sample(few, u, mask=one, k=2)
    check_sample(few, u, mask=one[0])


def test_sample_logits_settings_per_row_strides_and_shapes():
    g = gen(77)
    n = 24
    t = [0.0, 0.5, 1.0, 2.0] * 6
    k = [0, 1, 7, 1000] * 6
    p = [1.0, 0.9, 0.5] * 8
    mp = [0.0, 0.05] * 12
    for v in (40, 700):
        wide = rn(g, n, 2 * v + 3)
        u = torch.rand(n, generator=g, device="cuda")
        check_sample(wide[:, :v], u, t, k, p, mp, rows=True)
        check_sample(wide[:, 3:3 + v].bfloat16(), u, t, k, p, mp, rows=True)
        m = torch.rand(n, 2 * v, generator=g, device="cuda") < 0.6
        check_sample(wide[:, v:2 * v], u, 1.0, 9, 0.8, 0.0, mask=m[:, 1:v + 1])
    a = ops.sample_logits(wide.view(4, 6, -1), u.view(4, 6), top_p=0.9)
    b = ops.sample_logits(wide, u, top_p=0.9)
    assert torch.equal(a[0].view(-1), b[0]) and torch.equal(a[1].view(-1), b[1])
    tok, lp = ops.sample_logits(torch.empty(0, 5, device="cuda"), torch.empty(0, device="cuda"))
    assert tok.shape == (0,) and lp.shape == (0,)
    tok, lp = ops.sample_logits(torch.zeros(7, device="cuda"), torch.tensor(0.5, device="cuda"))
    assert tok.shape == () and int(tok) == 3


@pytest.mark.parametrize("n,v,dtype", [(1, 32001, torch.float32), (2, 131072, torch.bfloat16), (200, 20000, torch.float32),
                                       (1, 700001, torch.float32)])
def test_sample_logits_long_rows(n, v, dtype):
    """Rows that a cluster shares, rows of one block, and rows that are longer than the cluster's shared memory."""
    g = gen(v)
    logits = (rn(g, n, v) * 2).to(dtype)
    u = torch.rand(n, generator=g, device="cuda")
    k, p = 1000, 0.9
    tok, lp = ops.sample_logits(logits, u, temperature=0.8, top_k=k, top_p=p)
    l = logits.float()
    m = l.max(-1, keepdim=True).values
    z = torch.where(l == m, 0.0, (l - m) * float(np.float32(1) / np.float32(0.8)))
    q = torch.exp(z).double().mul(2.0 ** 40).long()
    order = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :k]
    qs = q.gather(1, order)
    before = qs.cumsum(-1) - qs
    keep = before.double() < float(np.float32(p)) * qs.sum(-1, keepdim=True).double()
    kept = torch.zeros_like(q).scatter_(1, order, torch.where(keep, qs, 0))
    run = kept.cumsum(-1)
    at = (u[:, None].double() * run[:, -1:].double()).long().minimum(run[:, -1:] - 1)
    want = (run > at).to(torch.uint8).argmax(-1)
    assert torch.equal(tok, want)
    ref = z.gather(1, want[:, None]).double()[:, 0] - torch.log(run[:, -1].double() / 2.0 ** 40)
    assert bool(((lp.double() - ref).abs() <= 2.0 ** -23 * (1 + ref.abs())).all())


def test_operators_on_another_stream():
    g = gen(9)
    x, w, h = rn(g, 4096, 512).bfloat16(), rn(g, 512).bfloat16(), rn(g, 4096, 512).bfloat16()
    ref = ops.block_norm(x, w, h)
    env = torch.arange(4096, device="cuda")
    dref = ops.counter_dropout(x, 0.5, 3, env)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x2 = x * 1.0                      # made on s, read on s
        y, n = ops.block_norm(x2, w, h)
        d = ops.counter_dropout(x2, 0.5, 3, env)
    s.synchronize()
    assert torch.equal(y, ref[0]) and torch.equal(n, ref[1]) and torch.equal(d, dref)


# ---------------------------------------------------------------------------------------------------- refusals
def test_refusals():
    x, w = torch.ones(4, 8, device="cuda"), torch.ones(8, device="cuda")
    env = torch.arange(4, device="cuda")
    U_, V, T = eng_mod.B200Unsupported, ValueError, TypeError
    bad = [
        (U_, lambda: ops.block_norm(x.cpu(), w)), (U_, lambda: ops.block_norm(x.double(), w.double())),
        (T, lambda: ops.block_norm(x, w.bfloat16())), (V, lambda: ops.block_norm(x, w[:4])),
        (V, lambda: ops.block_norm(x, w, gate=w)), (V, lambda: ops.block_norm(x, w, x[:2])),
        (V, lambda: ops.block_norm(x, w, x, gate=torch.ones(3, 8, device="cuda"))),
        (V, lambda: ops.block_norm(x, w, x, gate=torch.ones(4, 1, device="cuda"))),
        (U_, lambda: ops.block_norm(torch.ones(1, 8193, device="cuda"), torch.ones(8193, device="cuda"))),
        (T, lambda: ops.block_norm([1.0], w)),
        (V, lambda: ops.counter_dropout(x, 1.5, 1, env)), (V, lambda: ops.counter_dropout(x, 0.5, -1, env)),
        (T, lambda: ops.counter_dropout(x, 0.5, 1, env.int())), (V, lambda: ops.counter_dropout(x, 0.5, 1, env[:3])),
        (V, lambda: ops.counter_dropout(x, math.nan, 1, env)), (U_, lambda: ops.counter_dropout(x.long(), 0.5, 1, env)),
        (V, lambda: ops.sample_logits(x, torch.ones(3, device="cuda"))),
        (T, lambda: ops.sample_logits(x, torch.ones(4, device="cuda").double())),
        (V, lambda: ops.sample_logits(x, w[:4], top_k=-1)), (V, lambda: ops.sample_logits(x, w[:4], top_p=-0.1)),
        (V, lambda: ops.sample_logits(x, w[:4], min_p=1.5)), (V, lambda: ops.sample_logits(x, w[:4], temperature=-1.0)),
        (V, lambda: ops.sample_logits(x, w[:4], mask=torch.ones(4, 7, dtype=torch.bool, device="cuda"))),
        (T, lambda: ops.sample_logits(x, w[:4], mask=torch.ones(4, 8, device="cuda"))),
        (V, lambda: ops.sample_logits(x, w[:4], top_p=torch.ones(3, device="cuda"))),
    ]
    for i, (kind, f) in enumerate(bad):
        with pytest.raises(kind):
            f()
            pytest.fail(f"case {i} was not refused")
