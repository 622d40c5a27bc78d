"""distill_loss against a plain form in 64 bits.

Tolerances, u = 2^-24: with Z the largest |z - m| of a row (z = logits / tau, and the same of the teacher's), a weight exp(z - m) is
off by 4u + 3 Z u, a sum of V of them by V u more; so is q relative, log q absolute, and the loss by tau^2 (that + 4 u Z);
p likewise with K.  A gradient is off by g tau (q + p) times those, and half a step of its type."""
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


def check(logits, teacher, index, tau=1.0, mask=None, g=None):
    """Loss and gradient of every row; returns them."""
    rows, v = logits.shape
    k = teacher.shape[1]
    leaf = logits.detach().requires_grad_(True)
    loss = ops.distill_loss(leaf, teacher, index, temperature=tau, mask=mask)
    g = torch.linspace(-1, 2, rows, device="cuda") if g is None else g
    grad, = torch.autograd.grad(loss, leaf, g)
    with torch.no_grad():
        assert torch.equal(ops.distill_loss(logits, teacher, index, temperature=tau, mask=mask), loss)
    assert loss.dtype == torch.float32 and grad.dtype == logits.dtype and grad.shape == logits.shape
    tau = float(torch.tensor(tau))
    z = logits.double() / tau
    ok = logits != -math.inf
    if mask is not None:
        ok = ok & mask
    at = index.clamp(0, v - 1)
    on = (index >= 0) & (index < v) & torch.gather(ok, 1, at) & (teacher != -math.inf) & ~teacher.isnan()
    live = on.any(-1)
    z = torch.where(ok, z, -math.inf)
    logq = z - torch.logsumexp(torch.where(live[:, None], z, 0.0), -1, keepdim=True)
    t = torch.where(on, teacher.double() / tau, -math.inf)
    logp = t - torch.logsumexp(torch.where(live[:, None], t, 0.0), -1, keepdim=True)
    p = torch.where(on, torch.exp(logp), 0.0)
    lq = torch.gather(logq, 1, at)
    want = torch.where(live, torch.where(p > 0, p * (logp - lq), 0.0).sum(-1), 0.0) * tau ** 2
    q = torch.where(live[:, None] & ok, torch.exp(logq), 0.0)
    dense = torch.zeros_like(q).scatter_add_(1, at, p)
    wgrad = (g.double() * tau)[:, None] * (q - dense)
    spread = torch.where(ok & live[:, None], z.amax(-1, keepdim=True) - z, 0.0).amax(-1)
    spread = torch.maximum(spread, torch.where(on, t.amax(-1, keepdim=True) - t, 0.0).amax(-1))
    used = torch.where(p > 0, lq.abs() + logp.abs(), 0.0).amax(-1)          # the largest logarithm the loss is made of
    rel = (4 + 3 * spread + v ** 0.5 * 4 + k + 8) * U
    bound = tau ** 2 * (2 * rel + (8 + k) * U * used) + 2.0 ** -23 * want.abs()
    err = (loss.detach().double() - want).abs()
    assert bool((err <= bound).all()), ("loss", float((err / bound).max()))
    half = torch.finfo(grad.dtype).eps / 2
    tiny = 2.0 ** -24 if grad.dtype == torch.float16 else 1e-37
    bound = (half + 4 * U) * wgrad.abs() + (g.double().abs() * tau)[:, None] * (q + dense) * rel[:, None] * 1.01 + tiny
    err = (grad.double() - wgrad).abs()
    assert bool((err <= bound).all()), ("grad", float((err / bound).max()), float(err.max()))
    assert bool((grad[~ok] == 0).all()) and bool((grad[~live] == 0).all()) and bool((loss[~live] == 0).all())
    return loss.detach(), grad


def case(g, rows, v, k, dtype, tdtype=None):
    logits = (rn(g, rows, v) * 2).to(dtype)
    top = torch.topk(logits.float() + rn(g, rows, v), k)
    return logits, top.values.to(tdtype or dtype), top.indices


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,v,k", [(1, 1, 1), (5, 2, 2), (9, 33, 8), (7, 100, 31), (3, 1023, 128), (4, 1024, 64), (3, 1025, 129),
                                      (2, 4097, 1024), (700, 47, 5), (5, 9001, 50), (1, 131072, 64), (3, 40003, 7), (300, 2500, 3)])
def test_distill_loss(rows, v, k, dtype):
    g = gen(v + k)
    logits, teacher, index = case(g, rows, v, k, dtype)
    for tau, masked in ((1.0, False), (2.0, True), (0.5, False)):
        mask = torch.rand(rows, v, generator=g, device="cuda") < 0.6 if masked else None
        idx = index.clone()
        if masked:
            idx[torch.rand(rows, k, generator=g, device="cuda") < 0.2] = -1
        check(logits, teacher, idx, tau, mask)
    check(logits, teacher.float(), index)
    check(logits, teacher.to(torch.float16), index, mask=torch.rand(v, generator=g, device="cuda") < 0.5)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", [40, 700, 5003, 33000])
def test_rows_without_entries_and_odd_values(v, dtype):
    """Nothing allowed, nothing listed, indices out of range, the same index again, infinities and NaN in masked and in listed
    places, logits of the type's lowest value."""
    g = gen(v)
    logits, teacher, index = case(g, 10, v, 6, dtype)
    mask = torch.ones(10, v, dtype=torch.bool, device="cuda")
    mask[0] = False
    index[1] = -1
    index[2] = torch.tensor([v, -2, v + 7, 1 << 40, -(1 << 40), 3], device="cuda")
    index[3] = index[3, 0]
    index[4, 3] = index[4, 1]
    logits[5, ::3] = -math.inf
    logits[6] = -math.inf
    mask[7, ::2] = False
    logits[7, ::4] = math.nan
    logits[7, 2::4] = math.inf
    teacher[8, :3] = torch.tensor([-math.inf, math.nan, 0.0])
    logits[9, :v // 2] = torch.finfo(dtype).min
    index[9] = v - 1 - torch.arange(6, device="cuda")
    check(logits, teacher, index, mask=mask)
    logits[0] = math.nan                              # a row that allows nothing stays 0
    logits[6] = math.nan
    mask[6] = False
    check(torch.where(mask | (torch.arange(10, device="cuda") == 7)[:, None], logits, 0.0).to(dtype), teacher, index, mask=mask)
    leaf = logits.requires_grad_(True)
    loss = ops.distill_loss(leaf, teacher, index, mask=mask)
    grad, = torch.autograd.grad(loss.sum(), leaf)
    assert bool((loss[[0, 6]] == 0).all()) and bool((grad[[0, 6]] == 0).all())
    bad = logits.detach().clone()
    bad[5, 1] = math.nan                              # a NaN that is allowed is not hidden
    mask[:] = True
    l = ops.distill_loss(bad, teacher, index, mask=mask)
    assert bool(l[5].isnan())


@pytest.mark.parametrize("dtype", DT)
def test_strides_and_starts(dtype):
    """Rows apart, rows that start on any element, masks and logits whose rows start differently, leading axes.  Where a row
    starts decides which thread adds which of its elements: its sum is off by (V / 256 + 16) u = 40 u and by its weights' 4 + 3 Z
    = 64 u (Z below 20), log q and log p by that and their own rounding, 8 u: below 120 u a row, 240 u = 1.5e-5 between two."""
    near = lambda p, q: bool(((p - q).abs() <= 1.5e-5 + torch.finfo(p.dtype).eps * p.abs()).all())
    g = gen(3)
    for rows, v, k in ((6, 45, 4), (5, 6007, 20)):
        wide, teacher, index = case(g, rows, v + 9, k, dtype)
        index = index % v
        mask = torch.rand(rows, v + 5, generator=g, device="cuda") < 0.7
        for o in (0, 1, 3, 8):
            a = check(wide[:, o:o + v], teacher, index, mask=mask[:, 1:1 + v])
            b = check(wide[:, o:o + v].contiguous(), teacher, index, mask=mask[:, 1:1 + v].contiguous())
            assert near(a[0], b[0])
        x = wide[:, :v].reshape(rows, 1, v).expand(rows, 3, v).requires_grad_(True)
        t3, i3 = (q[:, None].expand(rows, 3, k) for q in (teacher, index))
        loss = ops.distill_loss(x, t3, i3)
        assert loss.shape == (rows, 3) and near(loss[:, 0], loss[:, 2])
        gr, = torch.autograd.grad(loss.sum(), x)
        assert gr.shape == x.shape and near(gr[:, 0], gr[:, 2])


def test_distill_gradient_against_differences():
    """fp32 logits, the loss summed in 64 bits: off by 2^-20 a row, over 2h = 2^-6; the third-order term is h^2."""
    g = gen(4)
    logits, teacher, index = case(g, 8, 300, 12, torch.float32)
    for tau in (1.0, 3.0):
        leaf = logits.detach().requires_grad_(True)
        f = lambda q: ops.distill_loss(q, teacher, index, temperature=tau).double().sum()
        grad, = torch.autograd.grad(f(leaf), leaf)
        way = rn(g, 8, 300)
        way /= way.norm()
        h = 2.0 ** -7
        with torch.no_grad():
            got = float((f(logits + h * way) - f(logits - h * way)) / (2 * h))
        want = float((grad.double() * way.double()).sum())
        assert abs(got - want) < 2.0 ** -9 * tau ** 2 * (1 + float(grad.norm()))


@pytest.mark.parametrize("v", [64, 65, 128, 129, 1024, 1025])
@pytest.mark.parametrize("k", [1, 7, 8, 9, 32, 33, 63, 64, 65, 128, 129, 255, 257])
def test_lists_of_every_form_with_repeated_entries(v, k):
    """Where the number of lanes of a row, and of entries that a lane holds, changes; odd lists; the same index many times."""
    g = gen(1000 * v + k)
    for dtype in DT:
        rows = 37
        logits = (rn(g, rows, v) * 2).to(dtype)
        index = torch.randint(-1, min(v, 40), (rows, k), generator=g, device="cuda")
        index[3] = v - 1
        check(logits, rn(g, rows, k).to(dtype), index, mask=torch.rand(rows, v, generator=g, device="cuda") < 0.8)


@pytest.mark.parametrize("rows,v,k", [(9600, 600, 5), (4800, 1000, 33), (4100, 2049, 9), (8200, 16384, 3), (2100, 400, 512), (1000, 400, 511),
                                      (740, 9000, 4), (370, 9000, 4)])
def test_many_rows_of_every_form(rows, v, k):
    """Where rows are many enough for a warp each, or few enough for several blocks each; rows apart and unaligned."""
    g = gen(rows)
    for dtype in (torch.bfloat16, torch.float32):
        wide = (rn(g, rows, v + 3) * 2).to(dtype)
        index = torch.randint(0, v, (rows, k), generator=g, device="cuda")
        check(wide[:, 1:1 + v], rn(g, rows, k).to(dtype), index)
