"""gated_ffn against its plain form in 64 bits, forward and backward, at sizes around the tiles and strides off 16 bytes.

Tolerances: y rounds h (F independent roundings of relative size U, taken up by the sum with weights wd) and itself; with
U the unit roundoff, the error of y is at most U |y| + U sum |h wd|, a bound the worst case over signs.  dx, dWg, dWu sum
rounded dg, du the same way; dWd sums rounded h.  fp32 accumulation of n products adds n 2^-24 of the sum of absolute
values, the activation's fast exponential 2^-20 of it.
"""
import importlib

import pytest
import torch

ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(n, d, f, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * n + d + f)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return (rn(n, d).to(dtype), (rn(f, d) * d ** -0.5).to(dtype), (rn(f, d) * d ** -0.5).to(dtype),
            (rn(d, f) * f ** -0.5).to(dtype), rn(n, d).to(dtype))


def act64(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = 0.5 * (1 + torch.erf(g / 2.0 ** 0.5))
    return g * c, c + g * torch.exp(-g * g / 2) * 0.3989422804014327


def reference(x, wg, wu, wd, dy, act):
    """(values, bounds' absolute sums) of y, dx, dwg, dwu, dwd in 64 bits."""
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    g, u = x @ wg.T, x @ wu.T
    a, da = act64(g, act)
    h, dh = a * u, dy @ wd
    dg, du = dh * u * da, dh * a
    vals = [h @ wd.T, dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ h]
    # what fp32 and the fast exponential leave in g, u, dh, a and da reaches dg and du in these absolute sizes
    gm, um, dm = x.abs() @ wg.abs().T, x.abs() @ wu.abs().T, dy.abs() @ wd.abs()
    hm, dgm, dum = (1 + gm) * um, dm * um * (1.2 + gm), dm * (1 + gm)
    tight = [h.abs() @ wd.abs().T, dg.abs() @ wg.abs() + du.abs() @ wu.abs(), dg.abs().T @ x.abs(), du.abs().T @ x.abs(),
             dy.abs().T @ h.abs()]
    loose = [hm @ wd.abs().T, dgm @ wg.abs() + dum @ wu.abs(), dgm.T @ x.abs(), dum.T @ x.abs(), dy.abs().T @ hm]
    return vals, tight, loose


def check(n, d, f, dtype, act, tensors=None):
    x, wg, wu, wd, dy = tensors or make(n, d, f, dtype)
    leaf = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = ops.gated_ffn(*leaf, act=act)
    got = [y.detach(), *torch.autograd.grad(y, leaf, dy)]
    vals, tight, loose = reference(x, wg, wu, wd, dy, act)
    u = U[dtype]
    tiny = 2.0 ** -24 * max(n, d, f) if dtype == torch.float16 else 1e-30      # fp16 subnormals of h, dg, du
    for name, a, v, t, l in zip(("y", "dx", "dw_gate", "dw_up", "dw_down"), got, vals, tight, loose):
        bound = u * v.abs() + u * t + (2.0 ** -20 + max(n, d, f) * 2.0 ** -24) * l + tiny
        err = (a.double() - v).abs()
        assert a.shape == v.shape and a.dtype == dtype
        assert bool((err <= bound).all()), f"{name}: worst {float((err / bound).max()):.2f} of the bound"
        rel = float(err.norm() / v.norm())
        assert rel <= 2 * u, f"{name}: relative error {rel:.2e}"
    with torch.no_grad():
        y2 = ops.gated_ffn(x, wg, wu, wd, act=act)
    near = (y2.double() - vals[0]).abs() <= u * vals[0].abs() + u * tight[0] + 2.0 ** -20 * loose[0] + tiny
    assert bool(near.all())
    assert ops.status() == 0
    return got


SHAPES = [(1, 8, 8), (1, 64, 128), (2, 16, 24), (3, 40, 72), (5, 7, 9), (16, 256, 512), (17, 100, 200), (33, 64, 96),
          (64, 128, 256), (127, 64, 130), (128, 128, 128), (129, 65, 129), (200, 512, 264), (257, 300, 500),
          (300, 1004, 681), (1000, 264, 1032), (2049, 136, 96), (1, 1, 1), (130, 1, 3), (1, 2000, 3001)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("n,d,f", SHAPES)
def test_gated_ffn_forward_and_backward(n, d, f, act, dtype):
    if (act == "gelu") != (dtype == torch.float16) and n * d * f > 10 ** 7:
        pytest.skip("each larger size once per type and activation")
    check(n, d, f, dtype, act)


def test_gated_ffn_more_tiles_than_sms_and_two_waves():
    check(4000, 520, 1160, torch.bfloat16, "silu")


def test_gated_ffn_strides_shapes_and_equal_bits():
    x, wg, wu, wd, dy = make(96, 128, 192, torch.bfloat16)
    a = check(96, 128, 192, torch.bfloat16, "silu", (x, wg, wu, wd, dy))
    b = check(96, 128, 192, torch.bfloat16, "silu", (x, wg, wu, wd, dy))
    for s, t in zip(a, b):
        assert torch.equal(s, t)                      # no sum depends on the order that blocks run in
    wide = torch.zeros(96, 400, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:136] = x
    wide[:, 201:329] = x
    for s in (wide[:, 8:136], wide[:, 201:329], x.t().contiguous().t()):
        assert torch.equal(ops.gated_ffn(s, wg, wu, wd), a[0])
    both = torch.cat((wg, wu))                        # one projection matrix, as two row ranges
    assert torch.equal(ops.gated_ffn(x, both[:192], both[192:], wd.t().contiguous().t()), a[0])
    assert torch.equal(ops.gated_ffn(x.view(8, 12, 128), wg, wu, wd).view(96, 128), a[0])
    assert torch.equal(ops.gated_ffn(x[0], wg, wu, wd), ops.gated_ffn(x[:1], wg, wu, wd)[0])


def test_gated_ffn_partial_gradients_empty_and_infinite():
    x, wg, wu, wd, dy = make(70, 64, 80, torch.bfloat16)
    full = check(70, 64, 80, torch.bfloat16, "silu", (x, wg, wu, wd, dy))
    for i in range(4):
        leaf = [t.detach().requires_grad_(j == i) for j, t in enumerate((x, wg, wu, wd))]
        y = ops.gated_ffn(*leaf)
        g, = torch.autograd.grad(y, leaf[i], dy)
        assert torch.equal(g, full[1 + i])
    leaf = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    g = torch.autograd.grad(ops.gated_ffn(*leaf).sum(), leaf)       # an expanded gradient
    g2 = torch.autograd.grad(ops.gated_ffn(*leaf), leaf, torch.ones_like(dy))
    assert all(torch.equal(s, t) for s, t in zip(g, g2))
    e = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    y = ops.gated_ffn(e, *leaf[1:])
    gr = torch.autograd.grad(y, [e, *leaf[1:]], torch.empty_like(y))
    assert y.shape == (0, 64) and not any(bool(t.any()) for t in gr[1:])
    bad = x.clone()
    bad[3, 5] = float("inf")
    bad[9, 0] = float("nan")
    y = ops.gated_ffn(bad, wg, wu, wd)
    ok = torch.ones(70, dtype=torch.bool, device="cuda")
    ok[[3, 9]] = False
    assert torch.equal(y[ok], full[0][ok]) and bool(y[9].isnan().all()) and not bool(y[3].isfinite().all())


def test_gated_ffn_gradient_against_differences():
    """Directional differences of the 64-bit scalar <y, dy> of fp16 outputs: the outputs' rounding (2^-11 of each, random) over
    the step bounds what the difference can show."""
    x, wg, wu, wd, dy = make(64, 96, 160, torch.float16)
    got = check(64, 96, 160, torch.float16, "gelu", (x, wg, wu, wd, dy))
    g = torch.Generator(device="cuda").manual_seed(8)
    base = [t.double() for t in (x, wg, wu, wd)]
    for i in range(4):
        step = 2.0 ** -3 * float(base[i].abs().mean())
        d = torch.sign(torch.randn(base[i].shape, generator=g, device="cuda")).double()
        f = []
        moved = []
        for s in (step, -step):
            t = [(b + s * d if j == i else b).half() for j, b in enumerate(base)]
            moved.append(t[i].double())
            f.append(float((ops.gated_ffn(*t, act="gelu").double() * dy.double()).sum()))
        want = float((got[1 + i].double() * (moved[0] - moved[1])).sum())
        size = float((got[1 + i].double().norm() * (moved[0] - moved[1]).norm()))
        assert abs(f[0] - f[1] - want) <= 0.02 * size


def test_gated_ffn_on_another_stream():
    x, wg, wu, wd, dy = make(300, 136, 200, torch.bfloat16)
    want = ops.gated_ffn(x, wg, wu, wd)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        y = ops.gated_ffn(x * 1.0, wg, wu, wd)
    s.synchronize()
    assert torch.equal(y, want)


def test_gated_ffn_refusals():
    x, wg, wu, wd, _ = make(4, 16, 24, torch.bfloat16)
    un, v, t = eng_mod.B200Unsupported, ValueError, TypeError
    bad = [(un, lambda: ops.gated_ffn(x.float(), wg.float(), wu.float(), wd.float())),
           (un, lambda: ops.gated_ffn(x.cpu(), wg, wu, wd)), (un, lambda: ops.gated_ffn(x, wg.cpu(), wu, wd)),
           (t, lambda: ops.gated_ffn(x, wg.half(), wu, wd)), (t, lambda: ops.gated_ffn(x, None, wu, wd)),
           (v, lambda: ops.gated_ffn(x, wg, wu, wd, act="tanh")), (v, lambda: ops.gated_ffn(x, wg, wu[:8], wd)),
           (v, lambda: ops.gated_ffn(x, wg, wu, wg)), (v, lambda: ops.gated_ffn(x[:, :8], wg, wu, wd)),
           (v, lambda: ops.gated_ffn(x, wg[0], wu, wd))]
    for i, (kind, f) in enumerate(bad):
        with pytest.raises(kind):
            f()
            pytest.fail(f"case {i} was not refused")
