"""The policy operators where sizes, sharing and autograd can go wrong: many rows, expanded inputs, saved tensors that change,
a second derivative, graphs, per-call state.  Tolerances as in the operators' own test files."""
import importlib
import math

import numpy as np
import pytest
import torch

ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu
DT = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


@pytest.mark.parametrize("n,d", [(200001, 8), (70000, 40), (1, 5000)])
def test_block_norm_many_rows(n, d):
    g = gen(n)
    x, h, w, p = rn(g, n, d), rn(g, n, d), rn(g, d), rn(g, d)
    leaf = [t.requires_grad_(True) for t in (x, h, w, p)]
    y, o = ops.block_norm(x, w, h, post_weight=p, scale=0.3)
    gy, gn = rn(g, n, d), rn(g, n, d)
    got = torch.autograd.grad((y, o), leaf, (gy, gn))
    l6 = [t.detach().double().requires_grad_(True) for t in leaf]
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    y6 = l6[0] + float(np.float32(0.3)) * (l6[3] * rms(l6[1]))
    o6 = l6[2] * rms(y6)
    ref = torch.autograd.grad((y6, o6), l6, (gy.double(), gn.double()))
    for a, b in zip((y, o, *got), (y6, o6, *ref)):
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) < 1e-5      # fp32 values and sums: 100 roundings of 2^-24


def test_gated_ffn_many_rows():
    """70001 rows: more m tiles than a grid has blocks, the last one with a single row."""
    g = gen(3)
    n, d, f = 70001, 64, 72
    x, dy = rn(g, n, d).bfloat16(), rn(g, n, d).bfloat16()
    wg, wu, wd = ((rn(g, *s) * s[1] ** -0.5).bfloat16() for s in ((f, d), (f, d), (d, f)))
    leaf = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = ops.gated_ffn(*leaf)
    got = [y, *torch.autograd.grad(y, leaf, dy)]
    l6 = [t.detach().double().requires_grad_(True) for t in leaf]
    y6 = (torch.nn.functional.silu(l6[0] @ l6[1].T) * (l6[0] @ l6[2].T)) @ l6[3].T
    ref = [y6, *torch.autograd.grad(y6, l6, dy.double())]
    for a, b in zip(got, ref):
        assert float((a.detach().double() - b.detach()).norm() / b.detach().norm()) < 2.0 ** -8      # three independent roundings of 2^-9 and less
    assert float((got[0].detach()[-1].double() - ref[0].detach()[-1]).norm() / ref[0].detach()[-1].norm()) < 2.0 ** -7


@pytest.mark.parametrize("n,v", [(300001, 5), (100000, 16), (40000, 40), (3000, 200)])
def test_sample_logits_many_rows(n, v):
    """Every row against the same definition in torch operations (fixed-point masses, stable sort)."""
    g = gen(v)
    l, u = rn(g, n, v) * 2, torch.rand(n, generator=g, device="cuda")
    mask = torch.rand(n, v, generator=g, device="cuda") < 0.8
    tok, lp = ops.sample_logits(l, u, top_k=max(2, v // 2), top_p=0.9, min_p=0.02, mask=mask)
    l = torch.where(mask, l, -math.inf)
    m = l.max(-1, keepdim=True).values
    dead = (m == -math.inf)[:, 0]
    z = torch.where(l == m, 0.0, l - m)
    w = torch.where(dead[:, None], 0.0, torch.exp(z))
    q = w.double().mul(2.0 ** 40).long()
    order = torch.sort(l, dim=-1, descending=True, stable=True).indices
    qs = q.gather(1, order)
    qs[:, max(2, v // 2):] = 0
    before = qs.cumsum(-1) - qs
    keep = before.double() < float(np.float32(0.9)) * qs.sum(-1, keepdim=True).double()
    keep[:, 0] = True
    q = torch.zeros_like(q).scatter_(1, order, torch.where(keep, qs, 0))
    q = torch.where(w >= np.float32(0.02).item(), q, 0)
    run = q.cumsum(-1)
    at = (u[:, None].double() * run[:, -1:].double()).long().minimum(run[:, -1:] - 1)
    want = torch.where(dead, -1, (run > at).to(torch.uint8).argmax(-1))
    assert torch.equal(tok, want) and bool((lp[dead] == -math.inf).all())


def test_expanded_inputs():
    g = gen(5)
    row, w = rn(g, 1, 48), rn(g, 48)
    x = row.expand(20, 48)
    assert torch.equal(ops.block_norm(x, w), ops.block_norm(x.contiguous(), w))
    leaf = row.clone().requires_grad_(True)
    a = torch.autograd.grad(ops.block_norm(leaf.expand(20, 48), w), leaf, torch.ones(20, 48, device="cuda"))[0]
    b = torch.autograd.grad(ops.block_norm(leaf, w), leaf, torch.ones(1, 48, device="cuda"))[0]
    assert torch.allclose(a, 20 * b, rtol=1e-5, atol=1e-5)
    mask = (torch.rand(1, 33, generator=g, device="cuda") < 0.5).expand(50, 33)
    l, u = rn(g, 50, 33), torch.rand(50, generator=g, device="cuda")
    assert torch.equal(ops.sample_logits(l, u, mask=mask)[0], ops.sample_logits(l, u, mask=mask.contiguous())[0])
    one = rn(g, 1, 33).expand(50, 33)
    assert torch.equal(ops.sample_logits(one, u)[0], ops.sample_logits(one.contiguous(), u)[0])
    x3 = rn(g, 6, 1, 32)[:, :, ::2].expand(6, 4, 16)             # neither rows of one stride nor whole elements
    assert torch.equal(ops.block_norm(x3, w[:16]), ops.block_norm(x3.contiguous(), w[:16]))
    x4 = rn(g, 7, 1, 40)[:, :, :16]                               # an axis of size 1 with a stride of its own
    assert torch.equal(ops.block_norm(x4, w[:16]), ops.block_norm(x4.contiguous(), w[:16]))
    gate = rn(g, 7, 1, 16)
    h = rn(g, 7, 5, 16)
    a = ops.block_norm(h, w[:16], h, gate=gate)
    b = ops.block_norm(h, w[:16], h, gate=gate.expand(7, 5, 16).contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_saved_tensors_that_change_and_second_derivatives():
    g = gen(6)
    x, w = rn(g, 12, 32).requires_grad_(True), rn(g, 32).requires_grad_(True)
    h = x * 1.0
    n = ops.block_norm(h, w)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError):                             # autograd notices
        n.sum().backward()
    n = ops.block_norm(x, w)
    gx, = torch.autograd.grad(n.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)
    xb = rn(g, 40, 32).bfloat16().requires_grad_(True)
    ws = [(rn(g, *s) * 0.2).bfloat16() for s in ((48, 32), (48, 32), (32, 48))]
    gx, = torch.autograd.grad(ops.gated_ffn(xb, *ws).float().square().sum(), xb, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.float().sum(), xb)
    env = torch.arange(12, device="cuda")
    gx, = torch.autograd.grad(ops.counter_dropout(x, 0.5, 1, env).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gx.sum(), x)


def test_graph_of_every_operator_replays():
    """One captured graph with a serving call (few rows), a larger forward call, norms, dropout and sampling: replays follow
    their inputs."""
    g = gen(7)
    x, big = rn(g, 6, 128).bfloat16(), rn(g, 300, 128).bfloat16()
    ws = [(rn(g, *s) * 0.1).bfloat16() for s in ((200, 128), (200, 128), (128, 200))]
    w = rn(g, 128).bfloat16()
    env = torch.arange(300, device="cuda")
    u = torch.rand(300, generator=g, device="cuda")

    def run():
        a = ops.gated_ffn(x, *ws)
        b = ops.gated_ffn(big, *ws)
        y, n = ops.block_norm(big, w, b, scale=0.5)
        d = ops.counter_dropout(n, 0.3, 5, env)
        t, lp = ops.sample_logits(d[:, :50], u, top_k=10, top_p=0.9)
        t2, _ = ops.sample_logits(d.float().view(1, -1), u[:1], top_k=100)
        return a, b, y, n, d, t, lp, t2

    run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for k in range(3):
        x.copy_(rn(g, 6, 128))
        big.copy_(rn(g, 300, 128))
        env.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, run()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 8, 9, 16, 17, 32, 33])
@pytest.mark.parametrize("d,f", [(8, 8), (24, 40), (250, 130), (1024, 512), (72, 3000), (3001, 72)])
def test_gated_ffn_few_rows(n, d, f, dtype):
    """The serving form around its row groups, odd widths (rows off 16 bytes) included; bounds as for the large form, with
    h unrounded up to 8 rows."""
    g = gen(n * d + f)
    x = rn(g, n, d).to(dtype)
    wg, wu, wd = ((rn(g, *s) * s[1] ** -0.5).to(dtype) for s in ((f, d), (f, d), (d, f)))
    y = ops.gated_ffn(x, wg, wu, wd, act="gelu")
    x6, g6, u6, d6 = (t.double() for t in (x, wg, wu, wd))
    gg = x6 @ g6.T
    h = gg * 0.5 * (1 + torch.erf(gg / 2.0 ** 0.5)) * (x6 @ u6.T)
    ref, mag = h @ d6.T, h.abs() @ d6.abs().T
    loose = ((1 + x6.abs() @ g6.abs().T) * (x6.abs() @ u6.abs().T)) @ d6.abs().T
    u = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
    bound = u * ref.abs() + (0.0 if n <= 8 else u) * mag + (2.0 ** -15 * mag if n <= 8 else 0.0) \
        + (2.0 ** -20 + max(d, f) * 2.0 ** -24) * loose + 2.0 ** -24 * max(d, f)
    err = (y.double() - ref).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


def test_sample_settings_of_wrong_types():
    l, u = torch.zeros(3, 4, device="cuda"), torch.zeros(3, device="cuda")
    for kw in (dict(temperature="1"), dict(top_k=None), dict(top_p=[0.9])):
        with pytest.raises(TypeError):
            ops.sample_logits(l, u, **kw)
    for kw in (dict(top_k=1.5), dict(temperature=math.nan), dict(top_p=math.nan), dict(min_p=-0.1)):
        with pytest.raises(ValueError):
            ops.sample_logits(l, u, **kw)
    with pytest.raises(TypeError):
        ops.sample_logits(l, u, top_p=torch.ones(3, device="cuda").half())
    assert int(ops.sample_logits(l, u, top_k=np.int64(2), temperature=np.float32(0.5))[0][0]) == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("v", [16, 47, 127, 130, 256, 257, 384, 385])
def test_sample_logits_of_rows_that_hardly_differ(v, dtype):
    """Rows whose logits all lie close together, are equal, or leave one another far behind, on both sides of each length
    at which the sampler changes its form; expectations as in test_sample_logits_filters."""
    from test_gpu_policy_ops import check_sample
    g = gen(3 * v)
    u = torch.rand(6, generator=g, device="cuda")
    near = rn(g, 6, v) * 1e-2
    steep = near.clone()
    steep[:, 0], steep[:, v // 2] = 60.0, 30.0
    steps = -torch.arange(v, device="cuda").float().expand(6, v) * 1e-6
    low = rn(g, 6, v) * 40
    mask = torch.rand(6, v, generator=g, device="cuda") < 0.5
    for logits in (near, steep, steps, low):
        for t, k, p, mp in ((1.0, 0, 0.95, 0.0), (1.5, v // 2, 0.6, 0.0), (0.01, 7, 1.0, 0.0), (1.0, v - 1, 0.99, 0.5)):
            check_sample(logits.to(dtype), u, t, k, p, mp)
            check_sample(logits.to(dtype), u, t, k, p, mp, mask=mask)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", [700, 4100, 20003])
def test_sample_logits_of_long_rows_that_hardly_differ(v, dtype):
    """The same for rows that a block or several share: equal logits, two values, infinities of both signs, masks."""
    from test_gpu_policy_ops import check_sample
    g = gen(7 * v)
    u = torch.rand(3, generator=g, device="cuda")
    near = rn(g, 3, v) * 1e-3
    holes = near.clone()
    holes[:, ::7], holes[0, 5] = -math.inf, math.nan
    high = near.clone()
    high[1:, 11::v // 3] = math.inf
    two = (near > 0).float()
    mask = torch.rand(3, v, generator=g, device="cuda") < 0.5
    for logits in (near, holes, high, two, two * 0.0 - 3.0):
        for t, k, p, mp in ((1.0, 0, 0.95, 0.0), (1.5, v // 2, 0.6, 0.0), (0.01, 50, 1.0, 0.3)):
            check_sample(logits.to(dtype), u, t, k, p, mp)
            check_sample(logits.to(dtype), u, t, k, p, mp, mask=mask)


@pytest.mark.parametrize("v", [1536, 1537, 4096, 4097])
@pytest.mark.parametrize("n", [2, 400])
def test_sample_logits_rows_do_not_depend_on_the_batch(n, v):
    """A row gives the same token and the same log-probability alone, in a few rows and in many, whatever form each takes."""
    g = gen(n + v)
    l, u = rn(g, n, v) * 2, torch.rand(n, generator=g, device="cuda")
    for kw in (dict(top_p=0.9), dict(top_k=300, top_p=0.8, temperature=1.3), dict(top_k=5), dict(min_p=0.01)):
        tok, lp = ops.sample_logits(l, u, **kw)
        for i in (0, 1, n // 2, n - 1):
            one, lp1 = ops.sample_logits(l[i:i + 1], u[i:i + 1], **kw)
            assert int(one) == int(tok[i]) and float(lp1) == float(lp[i])
