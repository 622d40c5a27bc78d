"""The policy's memory (causal_conv, selective_scan, their steps) against plain loops in 64 bits.

Tolerances.  u = 2^-24.  An output is off by half a step of its type, plus what fp32 loses on the way: K u times its
magnitude, the same formula with every term's absolute value.
conv: a sum of K + 1 products, each rounded once, then silu: sigmoid's exponential is off by 2 ulp = 4u and its argument's rounding
2 |p| u, the reciprocal 2u, two roundings: (K + 10 + 3 max|p|) u; a gradient is such a product again, and a sum over n elements
adds n u.
scan: delta is off by (14 + 3 max|v|) u relative (v rounded, exponential, reciprocal, series, sum), one decay by
4u + |delta a| (16 + 3 max|v|) u, and a path through T steps multiplies T decays forward and T backward and rounds twice a
step; the sums over N states, C channels or S T steps add as many u."""
import importlib
import math

import pytest
import torch

ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


def near(got, want, mag, k, name=""):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0          # fp16's smallest step, half of it twice
    half = torch.finfo(got.dtype).eps / 2
    bound = half * want.abs() + (1 + half) * k * U * mag + tiny + 1e-37
    err = (got.double() - want).abs()
    assert bool((err <= bound).all()), (name, float((err / bound).max()), float(err.max()))


def silu6(v):
    s = torch.sigmoid(v)
    return v * s, s * (1 + v * (1 - s))


# ------------------------------------------------------------------------------------------------- references
def spread(reset, lead, t):
    """reset [..., T] over x's leading sizes, as [S, T]; None: no flag."""
    if reset is None:
        return torch.zeros(math.prod(lead), t, dtype=torch.bool, device="cuda")
    r = reset.reshape((1,) * (len(lead) + 1 - reset.dim()) + tuple(reset.shape))
    return r.expand(*lead, t).reshape(-1, t)


def conv_ref(x, w, bias, state, reset, act, gy, gs, mag=False):
    """x [S, T, C] ...: y, state, and the gradients of x, w, bias, state for those (gy, gs) of the results."""
    s, t, c = x.shape
    k = w.shape[1]
    xp = torch.cat((state, x), 1)
    since = torch.full((s,), k - 1, device="cuda")
    valid = []
    for i in range(t):
        since = torch.where(reset[:, i], 0, since)
        valid.append(since.clone())
        since = since + 1
    valid = torch.stack(valid, 1) if t else torch.zeros(s, 0, device="cuda", dtype=torch.long)
    tap = [torch.where((valid >= j)[..., None], xp[:, k - 1 - j:k - 1 - j + t], 0.0) for j in range(k)]
    pre = bias + sum(w[:, k - 1 - j] * tap[j] for j in range(k))
    y, slope = silu6(pre) if act else (pre, torch.ones_like(pre))
    left = torch.stack([since >= k - 1 - i for i in range(k - 1)], 1)[..., None]        # entry i is k - 1 - i steps back
    new = torch.where(left, xp[:, t:], 0.0)
    if mag:
        ap, aw, at = xp.abs(), w.abs(), [v.abs() for v in tap]
        y = (bias.abs() + sum(aw[:, k - 1 - j] * at[j] for j in range(k))) * (1.2 if act else 1.0)
        g, w, tap, xp = gy.abs() * (1.2 + pre.abs() if act else 1.0), aw, at, ap
        gs = gs.abs()
        # a pre-activation that is off moves the slope, whose derivative is at most 1/2
        if act:
            g = g + 0.5 * gy.abs() * y
    else:
        g = gy * slope
    gx = torch.zeros_like(xp)
    for j in range(k):
        gx[:, k - 1 - j:k - 1 - j + t] += torch.where((valid >= j)[..., None], g * w[:, k - 1 - j], 0.0)
    gx[:, t:] += torch.where(left, gs, 0.0)
    gw = torch.stack([(g * tap[k - 1 - i]).sum((0, 1)) for i in range(k)], -1)
    return y, new, gx[:, k - 1:], gw, g.sum((0, 1)), gx[:, :k - 1], pre


def scan_ref(x, dt, a, b, c, d, z, bias, state, reset, gy, gs, mag=False):
    """y, state, and the gradients of x, dt, a, b, c, d, z, bias, state."""
    s, t, ch = x.shape
    v = dt + bias
    delta = torch.where(v > 0, v, 0.0) + torch.log1p(torch.exp(-v.abs()))
    sig = torch.sigmoid(v)
    sz, dz = silu6(z) if z is not None else (torch.ones_like(x), None)
    e = torch.exp(delta[..., None] * a)
    if mag:
        x, b, c, d, a, gy, gs, state, sz = (q.abs() for q in (x, b, c, d, a, gy, gs, state, sz))
        dz = dz.abs() + 0.5 if dz is not None else None
    g = gy * sz
    h, hs, before, ys = state, [], [], []
    for i in range(t):
        h = torch.where(reset[:, i, None, None], 0.0, h)
        before.append(h)
        h = e[:, i] * h + (delta[:, i] * x[:, i])[..., None] * b[:, i, None]
        hs.append(h)
        ys.append(torch.einsum("scn,sn->sc", h, c[:, i]) + d * x[:, i])
    new, y0 = h, torch.stack(ys, 1)
    r = gs
    gx, gdt, gb, gc = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(b), torch.zeros_like(c)
    ga = torch.zeros_like(a)
    for i in range(t - 1, -1, -1):
        dh = r + c[:, i, None] * g[:, i, :, None]
        q = dh * e[:, i] * before[i]
        s1 = torch.einsum("scn,sn->sc", dh, b[:, i])
        gx[:, i] = s1 * delta[:, i] + d * g[:, i]
        gdt[:, i] = (torch.einsum("scn,cn->sc", q, a) + s1 * x[:, i]) * sig[:, i]
        gb[:, i] = torch.einsum("scn,sc->sn", dh, delta[:, i] * x[:, i])
        gc[:, i] = torch.einsum("scn,sc->sn", hs[i], g[:, i])
        ga += torch.einsum("scn,sc->cn", q, delta[:, i])
        r = torch.where(reset[:, i, None, None], 0.0, e[:, i] * dh)
    return dict(y=y0 * sz, new=new, x=gx, dt=gdt, a=ga, b=gb, c=gc, d=(g * x).sum((0, 1)), z=gy * dz * y0 if dz is not None else None,
                dt_bias=gdt.sum((0, 1)), state=r, v=v, far=(delta[..., None] * a.abs()).amax())


# ------------------------------------------------------------------------------------------------- conv
def major(t, time):
    """The same values [E, R, T, ...], lying step by step."""
    return t.permute(2, 0, 1, *range(3, t.dim())).contiguous().permute(1, 2, 0, *range(3, t.dim())) if time else t


def conv_case(g, e, r, t, c, k, dtype, time=False, resets=0.0, env=True, carry=True, bias=True):
    x = major(rn(g, e, r, t, c).to(dtype), time)
    w, b = rn(g, c, k).to(dtype), rn(g, c).to(dtype) if bias else None
    state = rn(g, e, r, k - 1, c).to(dtype) if carry else None
    flags = torch.rand(e, 1 if env else r, t, generator=g, device="cuda") < resets if resets else None
    return x, w, b, state, flags


def check_conv(g, x, w, b, state, flags, act, through=True):
    e, r, t, c = x.shape
    k, dtype = w.shape[1], x.dtype
    leaf = [v.detach().requires_grad_(True) if v is not None else None for v in (x, w, b, state)]
    y, new = ops.causal_conv(*leaf[:3], state=leaf[3], reset=flags, act=act)
    assert y.dtype == new.dtype == dtype and new.shape == (e, r, k - 1, c)
    gy = rn(g, e, r, t, c).to(dtype)
    gs = rn(g, e, r, k - 1, c).to(dtype) if through else None
    wrt = [v for v in leaf if v is not None]
    got = torch.autograd.grad((y, new) if through else (y,), wrt, (gy, gs) if through else (gy,))
    f = lambda v, last: v.detach().double().reshape(-1, last, c)
    zero = torch.zeros(e * r, k - 1, c, dtype=torch.float64, device="cuda")
    args = (f(x, t), w.double(), b.double() if b is not None else torch.zeros(c, dtype=torch.float64, device="cuda"),
            f(state, k - 1) if state is not None else zero, spread(flags, (e, r), t), act, f(gy, t), f(gs, k - 1) if through else zero)
    want, mag = conv_ref(*args), conv_ref(*args, mag=True)
    n = k + 10 + 3 * float(want[6].abs().max()) + 2
    near(y.detach().reshape(-1, t, c), want[0], mag[0], n, "y")
    assert torch.equal(new.detach().double().reshape(-1, k - 1, c), want[1])
    total = e * r * t
    shapes = {"x": (2, (e * r, t, c), n), "w": (3, (c, k), n + total), "bias": (4, (c,), n + total), "state": (5, (e * r, k - 1, c), n)}
    it = iter(got)
    for v, name in zip(leaf, shapes):
        if v is not None:
            at, shape, m = shapes[name]
            near(next(it).reshape(shape), want[at], mag[at], m, name)
    with torch.no_grad():
        y2, new2 = ops.causal_conv(x, w, b, state=state, reset=flags, act=act)
    assert torch.equal(y2, y) and torch.equal(new2, new)
    return y.detach(), new.detach()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("k", [2, 3, 4])
@pytest.mark.parametrize("t,c", [(1, 8), (2, 5), (3, 64), (4, 33), (5, 260), (16, 4), (17, 100), (50, 1)])
def test_causal_conv(t, c, k, dtype):
    g = gen(t * 1000 + c * 10 + k)
    for time, resets, env, carry, bias, act in ((False, 0.0, True, False, True, "silu"), (True, 0.3, True, True, True, "silu"),
                                                (False, 0.3, False, True, False, None), (True, 1.0, True, True, True, "silu")):
        check_conv(g, *conv_case(g, 3, 2, t, c, k, dtype, time, resets, env, carry, bias), act)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("e,r,t,c", [(1, 1, 1000, 64), (1, 1, 4001, 12), (2, 1, 333, 1030), (700, 3, 9, 16)])
def test_causal_conv_split_over_time_and_over_many_tasks(e, r, t, c, dtype):
    """Parts of the time axis, their edges and a last part shorter than the taps; more sequences than workers."""
    g = gen(t + c)
    for resets in (0.0, 0.1):
        check_conv(g, *conv_case(g, e, r, t, c, 4, dtype, False, resets), "silu", through=resets > 0)


# ------------------------------------------------------------------------------------------------- scan
NAMES = ("x", "dt", "a", "b", "c", "d", "z", "dt_bias", "state")


def scan_case(g, e, r, t, ch, n, dtype, time=False, resets=0.0, env=True, carry=True, gate=True, plain=False):
    mk = lambda *s: major(rn(g, e, r, t, *s).to(dtype), time)
    bc = mk(2 * n)
    v = dict(x=mk(ch), dt=mk(ch), a=-torch.rand(ch, n, generator=g, device="cuda") * 3, b=bc[..., :n], c=bc[..., n:],
             d=None if plain else rn(g, ch), z=mk(ch) if gate else None, dt_bias=None if plain else rn(g, ch) - 2,
             state=rn(g, e, r, ch, n) if carry else None)
    flags = torch.rand(e, 1 if env else r, t, generator=g, device="cuda") < resets if resets else None
    return v, flags


def scan_call(v, flags):
    return ops.selective_scan(v["x"], v["dt"], v["a"], v["b"], v["c"], d=v["d"], z=v["z"], dt_bias=v["dt_bias"], state=v["state"],
                              reset=flags)


def scan_refs(v, flags, gy, gs):
    e, r, t, ch = v["x"].shape
    n = v["a"].shape[1]
    f = lambda q, *last: q.detach().double().reshape(-1, *last)
    zero = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")
    args = (f(v["x"], t, ch), f(v["dt"], t, ch), v["a"].detach().double(), f(v["b"], t, n), f(v["c"], t, n),
            v["d"].detach().double() if v["d"] is not None else zero(ch), f(v["z"], t, ch) if v["z"] is not None else None,
            v["dt_bias"].detach().double() if v["dt_bias"] is not None else zero(ch),
            f(v["state"], ch, n) if v["state"] is not None else zero(e * r, ch, n), spread(flags, (e, r), t), f(gy, t, ch),
            f(gs, ch, n) if gs is not None else zero(e * r, ch, n))
    return scan_ref(*args), scan_ref(*args, mag=True)


def check_scan(g, v, flags, through=True):
    e, r, t, ch = v["x"].shape
    n, dtype = v["a"].shape[1], v["x"].dtype
    leaf = {k: q.detach().requires_grad_(True) if q is not None else None for k, q in v.items()}
    y, new = scan_call(leaf, flags)
    assert y.dtype == dtype and new.dtype == torch.float32 and new.shape == (e, r, ch, n)
    gy = rn(g, e, r, t, ch).to(dtype)
    gs = rn(g, e, r, ch, n) if through else None
    wrt = [k for k in NAMES if leaf[k] is not None]
    got = torch.autograd.grad((y, new) if through else (y,), [leaf[k] for k in wrt], (gy, gs) if through else (gy,))
    want, mag = scan_refs(v, flags, gy, gs)
    vmax, far = float(want["v"].abs().max()), float(want["far"])
    step = 4 + far * (16 + 3 * vmax) + 2
    k = 2 * t * step + 2 * (14 + 3 * vmax) + n + 20 + 3 * (float(v["z"].abs().max()) if v["z"] is not None else 0)
    near(y.detach().reshape(-1, t, ch), want["y"], mag["y"], k, "y")
    near(new.detach().reshape(-1, ch, n), want["new"], mag["new"], k, "new")
    total = e * r * t
    for name, o in zip(wrt, got):
        assert o.shape == v[name].shape and o.dtype == v[name].dtype
        m = k + (ch if name in "bc" else total if name in ("a", "d", "dt_bias") else 0)
        near(o.reshape(want[name].shape), want[name], mag[name], m, name)
    with torch.no_grad():
        y2, new2 = scan_call(v, flags)
    assert torch.equal(y2, y) and torch.equal(new2, new)
    return got


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [1, 4, 5, 8, 10, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("t,ch", [(1, 7), (2, 40), (8, 33), (9, 1), (25, 130)])
def test_selective_scan(t, ch, n, dtype):
    g = gen(t * 1000 + ch * 10 + n)
    for time, resets, env, carry, gate, plain in ((False, 0.0, True, False, False, True), (True, 0.3, True, True, True, False),
                                                  (False, 0.2, False, True, True, False), (True, 1.0, True, True, False, False)):
        check_scan(g, *scan_case(g, 2, 2, t, ch, n, dtype, time, resets, env, carry, gate, plain))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("e,r,t,ch,n", [(1, 1, 300, 48, 16), (1, 1, 1001, 20, 5), (2, 1, 129, 700, 16), (300, 3, 11, 40, 16),
                                        (1, 2, 200, 24, 64), (1, 1, 260, 600, 3)])
def test_selective_scan_split_over_time_and_over_many_tasks(e, r, t, ch, n, dtype):
    """Parts of the time axis with and without an episode's start inside, several blocks over the channels, more sequences
    than workers."""
    g = gen(t + ch + n)
    for resets in (0.0, 0.02):
        check_scan(g, *scan_case(g, e, r, t, ch, n, dtype, False, resets), through=resets > 0)


# ------------------------------------------------------------------------------------------------- steps
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("e,r,c", [(1, 1, 1), (3, 5, 33), (2, 16, 260)])
def test_steps_equal_the_rollout(e, r, c, dtype):
    """Step by step with resets: conv's outputs and states have the rollout's bits; the scan's are near its (its states are
    rounded alike, its sums over states in another order)."""
    g = gen(c)
    t = 7
    for k, n in ((2, 4), (4, 16), (3, 10), (4, 64)):
        x, w, b, state, flags = conv_case(g, e, r, t, c, k, dtype, resets=0.3)
        with torch.no_grad():
            y, new = ops.causal_conv(x, w, b, state=state, reset=flags)
            live = state.clone()
            for i in range(t):
                o = ops.causal_conv_step(x[:, :, i], w, live, b, reset=flags[..., i])
                assert torch.equal(o, y[:, :, i])
            assert torch.equal(live, new)
        v, flags = scan_case(g, e, r, t, c, n, dtype, resets=0.3)
        live = v["state"].clone()
        gy = torch.zeros(e, r, t, c, device="cuda")
        want, mag = scan_refs(v, flags, gy, None)
        vmax, far = float(want["v"].abs().max()), float(want["far"])
        lim = 2 * t * (6 + far * (16 + 3 * vmax)) + 2 * (14 + 3 * vmax) + n + 20 + 3 * float(v["z"].abs().max())
        for i in range(t):
            at = lambda q: v[q][:, :, i]
            o = ops.selective_scan_step(at("x"), at("dt"), v["a"], at("b"), at("c"), live, d=v["d"], z=at("z"), dt_bias=v["dt_bias"],
                                        reset=flags[..., i])
            near(o.reshape(-1, c), want["y"][:, i], mag["y"][:, i], lim, "y")
        near(live.reshape(-1, c, n), want["new"], mag["new"], lim, "state")


def test_rollout_in_two_halves_equals_the_whole():
    """The state carries everything: two calls, and their gradients through the state, equal one call's (the memory's to its
    tolerance, whose parts may differ)."""
    g = gen(5)
    v, flags = scan_case(g, 2, 3, 24, 36, 16, torch.float32, resets=0.1)
    x, w, b, state, _ = conv_case(g, 2, 3, 24, 36, 4, torch.float32)
    leaf = [q.requires_grad_(True) for q in (x, w, b, state)]
    y, new = ops.causal_conv(*leaf[:3], state=leaf[3], reset=flags)
    one = torch.autograd.grad(y.square().sum() + new.sum(), leaf)
    y1, s1 = ops.causal_conv(leaf[0][:, :, :9], *leaf[1:3], state=leaf[3], reset=flags[..., :9])
    y2, s2 = ops.causal_conv(leaf[0][:, :, 9:], *leaf[1:3], state=s1, reset=flags[..., 9:])
    assert torch.equal(torch.cat((y1, y2), 2), y) and torch.equal(s2, new)
    two = torch.autograd.grad(y1.square().sum() + y2.square().sum() + s2.sum(), leaf)
    for p, q in zip(one, two):
        assert float((p - q).norm() / p.norm()) < 1e-6
    leaf = {k: q.requires_grad_(True) for k, q in v.items()}
    y, new = scan_call(leaf, flags)
    one = torch.autograd.grad(y.square().sum() + new.sum(), list(leaf.values()))
    cut = lambda p, q: {k: t[:, :, p:q] if k in ("x", "dt", "b", "c", "z") else t for k, t in leaf.items()}
    y1, s1 = scan_call(cut(0, 9), flags[..., :9])
    y2, s2 = scan_call({**cut(9, 24), "state": s1}, flags[..., 9:])
    two = torch.autograd.grad(y1.square().sum() + y2.square().sum() + s2.sum(), list(leaf.values()))
    for p, q in zip(one, two):
        assert float((p - q).norm() / p.norm()) < 1e-5


def test_gradients_against_differences():
    """Along a direction, in fp32 inputs: (f(p + hq) - f(p - hq)) / 2h with the loss summed in 64 bits from the operators' fp32
    outputs.  An output is off by about 2^-20, so is a difference of two over 2h = 2^-6: 2^-14 of the loss's size; the
    third-order term is h^2 = 2^-14 of it."""
    g = gen(11)
    v, flags = scan_case(g, 2, 1, 13, 8, 4, torch.float32, resets=0.2)
    wy, ws = rn(g, 2, 1, 13, 8).double(), rn(g, 2, 1, 8, 4).double()

    def loss(p):
        y, new = scan_call(p, flags)
        return (y.double() * wy).sum() + (new.double() * ws).sum()

    leaf = {k: q.detach().requires_grad_(True) for k, q in v.items()}
    grads = dict(zip(leaf, torch.autograd.grad(loss(leaf), list(leaf.values()))))
    for k, q in v.items():
        way = rn(g, *q.shape)
        way /= way.norm()
        h = 2.0 ** -7
        with torch.no_grad():
            got = float((loss({**v, k: q + h * way}) - loss({**v, k: q - h * way})) / (2 * h))
        want = float((grads[k].double() * way.double()).sum())
        assert abs(got - want) < 2.0 ** -10 * (1 + float(grads[k].norm())), (k, got, want)
    x, w, b, state, _ = conv_case(g, 2, 1, 13, 8, 4, torch.float32)
    vals = dict(x=x, w=w, b=b, state=state)

    def closs(p):
        y, new = ops.causal_conv(p["x"], p["w"], p["b"], state=p["state"], reset=flags)
        return (y.double() * wy).sum() + new.double().sum()

    leaf = {k: q.detach().requires_grad_(True) for k, q in vals.items()}
    grads = dict(zip(leaf, torch.autograd.grad(closs(leaf), list(leaf.values()))))
    for k, q in vals.items():
        way = rn(g, *q.shape)
        way /= way.norm()
        h = 2.0 ** -7
        with torch.no_grad():
            got = float((closs({**vals, k: q + h * way}) - closs({**vals, k: q - h * way})) / (2 * h))
        want = float((grads[k].double() * way.double()).sum())
        assert abs(got - want) < 2.0 ** -10 * (1 + float(grads[k].norm())), (k, got, want)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("k", [2, 3, 4])
@pytest.mark.parametrize("c,off", [(2, 0), (6, 0), (6, 2), (10, 1), (130, 0), (258, 4), (457, 0), (460, 0), (460, 3), (464, 2), (464, 4)])
def test_causal_conv_of_every_alignment(c, off, k, dtype):
    """Rows by 16, 8 and 4 bytes and by elements: even and odd widths, views off the boundary, time in parts."""
    g = gen(10 * c + off)
    for e, r, t in ((3, 2, 19), (1, 1, 150)):
        x, w, b, state, flags = conv_case(g, e, r, t, c, k, dtype, resets=0.1)
        wide = torch.zeros(e, r, t, c + 2 * off, device="cuda", dtype=dtype)
        wide[..., off:off + c] = x
        check_conv(g, wide[..., off:off + c], w, b, state, flags, "silu")
        with torch.no_grad():
            y, new = ops.causal_conv(x, w, b, state=state, reset=flags)
            live = state.clone()
            for i in range(t if t < 20 else 0):
                at = wide[:, :, i, off:off + c]
                near(ops.causal_conv_step(at, w, live, b, reset=flags[..., i]), y[:, :, i].double(), y[:, :, i].double().abs() + 16, 60)
            assert t > 19 or torch.equal(live, new)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("e,r,env", [(1, 1, True), (37, 3, True), (300, 1, False), (1, 500, True), (2500, 16, True)])
@pytest.mark.parametrize("c,n", [(1, 1), (1, 64), (3, 5), (18, 4), (40, 16), (33, 10), (129, 4)])
def test_scan_steps_of_few_channels(e, r, env, c, n, dtype):
    """A block takes several sequences side by side: every one of them, its own flag, and nothing behind the last."""
    g = gen(e + c + n)
    v, flags = scan_case(g, e, r, 1, c, n, dtype, resets=0.3, env=env)
    want, mag = scan_refs(v, flags, torch.zeros(e, r, 1, c, device="cuda"), None)
    vmax, far = float(want["v"].abs().max()), float(want["far"])
    lim = 2 * (6 + far * (16 + 3 * vmax)) + 2 * (14 + 3 * vmax) + n + 20 + 3 * float(v["z"].abs().max())
    room = torch.full((e * r + 7, c, n), 5.0, device="cuda")
    live = room[:e * r].view(e, r, c, n).copy_(v["state"])
    at = lambda q: v[q][:, :, 0]
    o = ops.selective_scan_step(at("x"), at("dt"), v["a"], at("b"), at("c"), live, d=v["d"], z=at("z"), dt_bias=v["dt_bias"], reset=flags[..., 0])
    near(o.reshape(-1, c), want["y"][:, 0], mag["y"][:, 0], lim, "y")
    near(live.reshape(-1, c, n), want["new"], mag["new"], lim, "state")
    assert bool((room[e * r:] == 5.0).all())


@pytest.mark.parametrize("e,r,t,ch,n", [(1, 3, 127, 377, 10), (1, 1, 64, 512, 16), (1, 16, 700, 200, 5), (2, 32, 130, 64, 64),
                                        (5, 16, 90, 300, 8), (1, 1, 33, 1024, 4)])
def test_selective_scan_where_parts_end_soonest(e, r, t, ch, n):
    """Forward and backward split in their own numbers of parts, down to parts of 16 steps."""
    g = gen(t + ch)
    for resets in (0.0, 0.05):
        check_scan(g, *scan_case(g, e, r, t, ch, n, torch.bfloat16, resets=resets))
