"""The policy operators where a fault of one tile, row or call could reach another.  Tolerances as in the operators' own
test files."""
import importlib
import math
import os
import subprocess
import sys

import pytest
import torch

ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DT = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


@pytest.mark.parametrize("n,d,f", [(60000, 96, 544),      # y and dx: N = 96, more pairs' tiles than pairs of SMs
                                   (64, 2080, 4640)])     # dWg, dWu (N = 2080) and dWd (N = 4640), their sums not split
def test_gated_ffn_edge_columns_of_many_tiles(n, d, f):
    """Widths that end 32 columns into a warp's 64: it sends one staged tile where it otherwise sends two, and goes on with
    another tile of the matrix.  Every element against 64 bits, and equal bits in a second call."""
    from test_gpu_policy_ffn import check
    first = check(n, d, f, torch.bfloat16, "silu")
    for _ in range(2):
        for a, b in zip(first, check(n, d, f, torch.bfloat16, "silu")):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", [385, 511, 1001, 1002, 1003, 1535, 4095])
def test_sample_logits_rows_that_end_inside_an_access(v, dtype):
    """Rows that a block keeps in shared memory, at every remainder of a 16-byte access: masked up to the last element, and
    with the last element alone."""
    from test_gpu_policy_ops import check_sample
    g = gen(v)
    logits, u = (rn(g, 5, v) * 2).to(dtype), torch.rand(5, generator=g, device="cuda")
    ends = torch.rand(5, v, generator=g, device="cuda") < 0.5
    ends[:, -1] = True
    last = torch.zeros(5, v, dtype=torch.bool, device="cuda")
    last[:, -1] = True
    for mask in (None, ends, last):
        for k, p in ((0, 0.9), (200, 0.8), (v - 1, 1.0)):
            check_sample(logits, u, 1.0, k, p, 0.0, mask=mask)


@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("d,dtype", [(5000, torch.float32), (8191, torch.float32), (8192, torch.float32), (6001, torch.bfloat16),
                                     *((d, t) for d in (1000, 1001) for t in DT)])
def test_block_norm_bad_rows_stay_alone(d, dtype, post):
    """Rows with a NaN or an infinity in x or h and a zero row without eps, among more rows than there are workers: every
    other row's outputs and gradients have the bits of the run without them."""
    g = gen(d)
    n, bad = 700, [5, 6, 300, 512]
    x, h, w, p = rn(g, n, d).to(dtype), rn(g, n, d).to(dtype), rn(g, d).to(dtype), rn(g, d).to(dtype)
    gy, gn = rn(g, n, d).to(dtype), rn(g, n, d).to(dtype)
    xb, hb = x.clone(), h.clone()
    xb[5, 3] = math.nan
    hb[6, d - 1] = math.inf
    xb[300], hb[300] = 0.0, 0.0
    hb[512, 0] = math.nan

    def run(x, h):
        leaf = [t.clone().requires_grad_(True) for t in (x, h)]
        y, o = ops.block_norm(leaf[0], w, leaf[1], post_weight=p if post else None, scale=0.5, eps=0.0)
        alone = ops.block_norm(x, w, eps=0.0)
        return [y.detach(), o.detach(), *torch.autograd.grad((y, o), leaf, (gy, gn)), alone]

    ok = torch.ones(n, dtype=torch.bool, device="cuda")
    ok[bad] = False
    got, want = run(xb, hb), run(x, h)
    for a, b in zip(got, want):
        assert bool(b.isfinite().all()) and torch.equal(a[ok], b[ok])
    assert bool(got[1][[5, 300, 512]].isnan().all()) and bool(got[4][[5, 300]].isnan().all())
    for i in (0, 5, 300, 301, 699):                 # a row does not depend on its place
        one = ops.block_norm(xb[i:i + 1], w, hb[i:i + 1], post_weight=p if post else None, scale=0.5, eps=0.0)
        for a, b in zip(one, got):
            assert torch.equal(a[0].view(torch.uint8), b[i].view(torch.uint8))


CAPTURED_FIRST = r"""
import ctypes, importlib, torch
nat = importlib.import_module("isaac-net_b200._native")
ops = importlib.import_module("isaac-net_b200.policy_ops")
seen = []


def entry(args, stream):                  # in place of the library's entry point: notes the word, launches nothing
    seen.append(args.contents.status)
    return 0


entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.POINTER(nat.InbFfnArgs), ctypes.c_void_p)(entry)
names = [*nat.POLICY_EXPORTS, "inb_block_norm_work", "inb_gated_ffn_work"]
at = {n: ctypes.cast(getattr(nat.lib(), n), ctypes.c_void_p).value for n in names}
at["inb_gated_ffn_fwd"] = ctypes.cast(entry, ctypes.c_void_p).value
ops._ext.bind(at, ValueError)
x, *w = (torch.zeros(s, device="cuda").bfloat16() for s in ((40, 16), (24, 16), (24, 16), (16, 24)))
a = torch.ones(3, device="cuda")
graph, streams = torch.cuda.CUDAGraph(), [torch.cuda.Stream() for _ in range(CYCLE)]
with torch.cuda.graph(graph, stream=streams[0] if streams else None):
    ops.gated_ffn(x, *w)
    b = a + 1
graph.replay()
assert b.tolist() == [2.0, 2.0, 2.0] and ops.status() == 0
del graph
ops.gated_ffn(x, *w)
assert seen[0] is not None and seen[0] == seen[1], seen
"""


@pytest.mark.parametrize("cycle", [0, 32])
def test_status_word_where_the_first_call_is_captured(cycle):
    """The first call of a process, made during a capture, passes the word that every later call passes.  32: torch hands its
    streams out in turn, and the next would be the one that is captured."""
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST.replace("CYCLE", str(cycle))], cwd=ROOT, capture_output=True,
                       text=True)
    assert r.returncode == 0, r.stderr


def test_status_waits_for_every_stream():
    g = gen(4)
    x, *w = (rn(g, *s).bfloat16() for s in ((40, 16), (24, 16), (24, 16), (16, 24)))
    ops.gated_ffn(x, *w)
    s, done = torch.cuda.Stream(), torch.cuda.Event()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(50_000_000)              # some 30 ms
        done.record()
    assert ops.status() == 0 and done.query()


@pytest.mark.parametrize("v", [5, 40, 130, 700, 3000, 20003])
def test_sample_logits_row_settings_out_of_range(v):
    """Per-row settings that are NaN or beyond their range count as 0 or as the nearest in range, in every form of the sampler."""
    g = gen(v)
    n = 8
    l, u = rn(g, n, v), torch.rand(n, generator=g, device="cuda")
    row = lambda value, dtype=torch.float32: torch.full((n,), value, dtype=dtype, device="cuda")
    same = [(dict(top_p=row(math.nan)), dict(top_p=0.0)), (dict(top_p=row(-2.0)), dict(top_p=0.0)),
            (dict(top_p=row(math.nan), top_k=min(v, 50)), dict(top_p=0.0)), (dict(top_p=row(1.5)), dict()),
            (dict(temperature=row(math.nan)), dict(temperature=0.0)), (dict(temperature=row(-1.0)), dict(temperature=0.0)),
            (dict(min_p=row(math.nan)), dict()), (dict(min_p=row(-1.0)), dict()), (dict(min_p=row(2.0)), dict(min_p=1.0)),
            (dict(top_k=row(-3, torch.int32)), dict()), (dict(top_k=row(v + 1, torch.int32)), dict())]
    for odd, plain in same:
        got, want = ops.sample_logits(l, u, **odd), ops.sample_logits(l, u, **plain)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), odd
    first = l.argmax(-1)
    for kw in (dict(top_p=row(math.nan)), dict(temperature=row(-1.0))):
        tok, logp = ops.sample_logits(l, u, **kw)
        assert torch.equal(tok, first) and not bool(logp.any())
    mixed = row(0.9)
    mixed[::2] = math.nan                          # among rows that are in range
    tok, _ = ops.sample_logits(l, u, top_p=mixed)
    assert torch.equal(tok[::2], first[::2]) and torch.equal(tok[1::2], ops.sample_logits(l, u, top_p=0.9)[0][1::2])


def test_forward_mode_is_refused():
    """A tangent, with and without reverse mode beside it, is refused and not dropped; a dual tensor without one is taken."""
    import torch.autograd.forward_ad as fwd
    g = gen(1)
    x, w = rn(g, 40, 32).bfloat16(), rn(g, 32).bfloat16()
    ws = [(rn(g, *s) * 0.2).bfloat16() for s in ((48, 32), (48, 32), (32, 48))]
    env, u = torch.arange(40, device="cuda"), torch.rand(40, generator=g, device="cuda")
    for grad, leaf in ((True, False), (True, True), (False, False)):
        with torch.set_grad_enabled(grad), fwd.dual_level():
            dual = lambda t: fwd.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t))
            d, dw, d0 = dual(x), dual(w), dual(ws[0])
            for f in (lambda: ops.block_norm(d, w), lambda: ops.block_norm(x, dw), lambda: ops.block_norm(x, w, d),
                      lambda: ops.block_norm(x, w, x, post_weight=dw), lambda: ops.block_norm(x, w, x, gate=d),
                      lambda: ops.gated_ffn(d, *ws), lambda: ops.gated_ffn(x, d0, *ws[1:]),
                      lambda: ops.counter_dropout(d, 0.5, 1, env), lambda: ops.sample_logits(d, u)):
                with pytest.raises(eng_mod.B200Unsupported, match="tangent"):
                    f()
            assert torch.equal(ops.block_norm(fwd.unpack_dual(d).primal, w).detach(), ops.block_norm(x, w))


@pytest.mark.parametrize("n", [4, 40, 300])
def test_gated_ffn_views_that_share_an_address_or_rows(n):
    """w_gate and w_up as views of one matrix that start at one address with different strides; x and a gradient whose rows
    overlap or are all one row.  Bits as on contiguous copies."""
    g = gen(n)
    x, dy, wd = rn(g, n, 64).bfloat16(), rn(g, n, 64).bfloat16(), (rn(g, 64, 96) * 0.2).bfloat16()
    w = (rn(g, 2 * 96, 64) * 0.2).bfloat16()

    def run(x, wg, wu, dy):
        leaf = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = ops.gated_ffn(*leaf)
        return [ops.gated_ffn(x, wg, wu, wd), y.detach(), *torch.autograd.grad(y, leaf, dy)]

    one, over = rn(g, 1, 64).bfloat16().expand(n, 64), torch.as_strided(rn(g, 64 + 8 * n).bfloat16(), (n, 64), (8, 1))
    for args in ((x, w[::2], w[:96], dy), (x, w[:96], w[::2], dy), (one, w[:96], w[96:], dy), (over, w[:96], w[96:], dy),
                 (x, w[:96], w[96:], one), (x, w[:96], w[:96], dy)):
        for a, b in zip(run(*args), run(*(t.contiguous() for t in args))):
            assert torch.equal(a, b)


def test_the_example_differentiates_what_it_sampled_from():
    """The log-probability that the policy gradient differentiates is the one that the sampler returned for its token.  Both
    come from the same fp32 logits by fewer than 16 roundings of 2^-24 of the largest number on the way."""
    from test_gpu_policy_loop import example
    ex = example()
    ib, presets = importlib.import_module("isaac-net_b200"), importlib.import_module("isaac-net_b200.presets")
    wl = presets.workload(1)
    net = ib.NetModule("L2", 8, 16, "cuda", wl.config(traffic=(), msg_sizes=(200.0, 1500.0, 8192.0)), seed=wl.seed,
                       isaac=ib.IsaacNetCfg(radio="engine", obs_features=("aoi", "sinr", "queue_len")))
    policy = ex.Policy(net.obs_dim, classes=4, seed=3)
    with torch.no_grad():
        policy.head.mul_(20)                       # probabilities that differ
    net.reset()
    obs = rn(gen(5), *net.obs().shape)
    for drop in (None, ex.step_key(net)):
        send, logp = ex.act(policy, net, obs, drop)
        again = ex.log_prob(policy, obs, send, drop)
        size = 1 + float(policy.logits(obs, drop).detach().abs().max())
        assert again.requires_grad and float((again.detach() - logp).abs().max()) <= 16 * 2.0 ** -24 * size
        assert float(logp.std()) > 0.1 and len(send.unique()) == 4


@pytest.mark.parametrize("dtype,tie", [(torch.float16, 2.0 ** -5), (torch.bfloat16, 2.0 ** -2)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("n", [1, 200])
def test_gated_ffn_keeps_projections_rounded(n, act, dtype, tie):
    """The projections kept for the backward pass are rounded to nearest.  g = |u| = 64 + tie + 5 2^-12, exact in fp32, where
    act(g) = g and act'(g) = 1: dg and du are the projections themselves (dh = 1), and lie 5 2^-12 above the middle of two
    numbers of the type.  24 bits hold 2^-9 of them: rounded they stay above it, cut they would fall onto it and go down."""
    x = torch.zeros(n, 8, dtype=dtype, device="cuda")
    x[0, :3] = torch.tensor([64.0, tie, 5 * 2.0 ** -12])
    wg = torch.zeros(24, 8, dtype=dtype, device="cuda")
    wg[:, :3] = 1.0
    wu, wd = wg.clone(), torch.zeros(8, 24, dtype=dtype, device="cuda")
    wu[12:] *= -1.0
    wd[0] = 1.0
    dy = torch.zeros(n, 8, dtype=dtype, device="cuda")
    dy[0, 0] = 1.0
    leaf = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    _, dwg, dwu, dwd = torch.autograd.grad(ops.gated_ffn(*leaf, act=act), leaf, dy)
    g = x.detach()[0].double().sum()
    up = g.to(dtype)
    assert float(up) == 64 + 2 * tie
    sign = torch.ones(24, 1, dtype=torch.float64, device="cuda")
    sign[12:] = -1.0
    row = x.detach()[0].double()
    assert torch.equal(dwg, (sign * up.double() * row).to(dtype))
    assert torch.equal(dwu, (up.double() * row).expand(24, 8).to(dtype))


def test_gated_ffn_keeps_nan_and_infinity_for_the_backward_pass():
    """Projections that are NaN (of either sign and any payload) or infinite reach the gradients as such, and only their own
    rows' dx."""
    g = gen(6)
    n, d, f = 70, 64, 80
    x, dy = rn(g, n, d).bfloat16(), rn(g, n, d).bfloat16()
    ws = [(rn(g, *s) * 0.2).bfloat16() for s in ((f, d), (f, d), (d, f))]
    bits = x.view(torch.int16)
    bits[3, 5], bits[9, 0], bits[20, 1], bits[21, 1] = 0x7FFF, -1, 0x7F80, -0x80        # NaN, -NaN, inf, -inf
    leaf = [t.detach().requires_grad_(True) for t in (x, *ws)]
    dx, = torch.autograd.grad(ops.gated_ffn(*leaf), leaf[:1], dy)
    ok = torch.ones(n, dtype=torch.bool, device="cuda")
    ok[[3, 9, 20, 21]] = False
    assert bool(dx[[3, 9]].isnan().all()) and not bool(dx[[20, 21]].isfinite().any()) and bool(dx[ok].isfinite().all())


def sample_rows(l, u, k, p, t, mask):
    """sample_logits' definition in torch operations, a row after another of up to millions of logits (k: 0 off; p: 1 off)."""
    l = torch.where(torch.isnan(l.float()), -math.inf, l.float())
    if mask is not None:
        l = torch.where(mask, l, -math.inf)
    inv = torch.tensor(1.0, device=l.device) / torch.tensor(t, device=l.device)
    tok, logp = [], []
    for row, r in zip(l, u):
        m = row.max()
        if m == -math.inf:
            tok.append(-1), logp.append(-math.inf)
            continue
        z = torch.where(row == m, 0.0, (row - m) * inv)
        q = torch.exp(z).double().mul(2.0 ** 40).long()
        order = torch.sort(row, descending=True, stable=True).indices
        qs = q[order]
        if k > 0:
            qs[k:] = 0
        if p < 1:
            before = qs.cumsum(0) - qs
            keep = before.double() < float(torch.tensor(p)) * qs.sum().double()
            keep[0] = True
            qs = torch.where(keep, qs, 0)
        run = torch.zeros_like(q).scatter_(0, order, qs).cumsum(0)
        at = min(int(float(r) * float(run[-1])), int(run[-1]) - 1)
        i = int((run > at).to(torch.uint8).argmax())
        tok.append(i), logp.append(float(z[i]) - math.log(int(run[-1]) / 2.0 ** 40))
    return torch.tensor(tok), torch.tensor(logp, dtype=torch.float64)


@pytest.mark.parametrize("n,v,dtype", [(3, 1000003, torch.bfloat16), (2, 1000001, torch.float16), (3, 450001, torch.float32),
                                       (64, 50257, torch.bfloat16), (200, 8193, torch.float16), (37, 20011, torch.float32)])
def test_sample_logits_long_rows_of_odd_length(n, v, dtype):
    """Rows beyond what eight blocks keep in shared memory, and batches of an odd vocabulary, whose rows start on every
    remainder of an access: with and without a mask, in rows of a wider matrix too, one row allowing nothing."""
    g = gen(v)
    wide = (rn(g, n, v + 3) * 2).to(dtype)
    wide[:, 7], wide[0, 11] = math.nan, -math.inf
    u = torch.rand(n, generator=g, device="cuda")
    some = torch.rand(n, v, generator=g, device="cuda") < 0.5
    some[n - 1] = False
    for l in (wide[:, 3:].contiguous(), wide[:, 1:v + 1]):
        for mask, k, p, t in ((None, 0, 0.9, 1.0), (some, 0, 0.95, 0.7), (some, 40, 0.9, 1.0), (None, 5000, 0.8, 1.5),
                              (some, 1, 1.0, 1.0), (some, 0, 1.0, 1.0)):
            tok, logp = ops.sample_logits(l, u, top_k=k, top_p=p, temperature=t, mask=mask)
            want, ref = sample_rows(l, u, k, p, t, mask)
            assert torch.equal(tok.cpu(), want)
            fin = torch.isfinite(ref)
            assert torch.equal(torch.isfinite(logp.cpu()), fin)
            assert bool(((logp.cpu().double() - ref)[fin].abs() <= 2.0 ** -23 * (1 + ref[fin].abs())).all())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("e,n", [(1500, 4095), (257, 20001), (3, 700003)])
def test_counter_dropout_large_batches_of_odd_rows(e, n, dtype):
    """Rows that start on every remainder of an access, forward and backward, against the hash in torch's 64-bit integers."""
    M = 0xFFFFFFFF
    p, s0 = 0.3, 77
    env = torch.arange(e, device="cuda") + 5

    def mix(v):
        v = v ^ (v >> 16)
        v = (v * 0x21F0AAAD) & M
        v = v ^ (v >> 15)
        v = (v * 0x735A2D97) & M
        return v ^ (v >> 15)

    salt = lambda w: (mix(w & M) + 0x9E3779B9) & M
    key = torch.full_like(env, s0)
    for word in (env, 0 * env, torch.full_like(env, 0x44), 0 * env, 0 * env):
        key = mix(key ^ salt(word))
    assert int(key[0]) == _host_key(s0, int(env[0]))
    j = torch.arange((n + 1) // 2, device="cuda") * 0x9E3779B9 & M
    x, gy = rn(gen(n), e, n).to(dtype).requires_grad_(True), rn(gen(e), e, n).to(dtype)
    y = ops.counter_dropout(x, p, s0, env)
    gx, = torch.autograd.grad(y, x, gy)
    threshold = round(p * 65536)
    for i in range(0, e, 64):
        w = mix(mix((key[i:i + 64, None] + j) & M) ^ key[i:i + 64, None])
        keep = torch.stack((w & 0xFFFF, w >> 16), -1).flatten(1)[:, :n] >= threshold
        for a, b in ((y, x), (gx, gy)):
            want = torch.where(keep, b[i:i + 64].detach().float() * (65536 / (65536 - threshold)), 0.0).to(dtype)
            assert torch.equal(a[i:i + 64].detach(), want)


def _host_key(s0, env):
    mix, salt = eng_mod._mix32, eng_mod._salt
    k = mix(s0 ^ salt(env))
    for v in (0, 0x44, 0, 0):
        k = mix(k ^ salt(v))
    return k


def big(rows, cols, dtype=torch.bfloat16):
    """Rows of a small random matrix over and over, 2^31 elements and more."""
    part = rn(gen(cols), 4099, cols).to(dtype)
    return part.repeat(-(-rows // 4099), 1)[:rows].contiguous()


def test_offsets_beyond_32_bits():
    """Tensors of more than 2^31 elements: their last rows have the bits that the same rows give alone."""
    n, d = 525000, 4096
    x, w = big(n, d), rn(gen(1), d).bfloat16()
    last = slice(n - 40, n)
    y, o = ops.block_norm(x, w, x, post_weight=w, scale=0.5)
    a, b = ops.block_norm(x[last], w, x[last], post_weight=w, scale=0.5)
    assert torch.equal(y[last], a) and torch.equal(o[last], b)
    del y, o
    leaf, part = x.requires_grad_(True), x.detach()[last].requires_grad_(True)
    gx, = torch.autograd.grad(ops.block_norm(leaf, w), leaf, x.detach())
    px, = torch.autograd.grad(ops.block_norm(part, w), part, part.detach())
    assert torch.equal(gx[last], px)
    del gx
    x = x.detach()
    env = torch.arange(n, device="cuda")
    assert torch.equal(ops.counter_dropout(x, 0.5, 1, env)[last], ops.counter_dropout(x[last], 0.5, 1, env[last]))
    u = torch.rand(n, generator=gen(2), device="cuda")
    mask = torch.ones(1, 1, dtype=torch.bool, device="cuda").expand(n, d)
    for v in (d, 33):                            # the short rows lie 4096 apart
        tok, logp = ops.sample_logits(x[:, :v], u, top_p=0.9, mask=mask[:, :v])
        t, p = ops.sample_logits(x[last, :v], u[last], top_p=0.9)
        assert torch.equal(tok[last], t) and torch.equal(logp[last], p)


def test_gated_ffn_offsets_beyond_32_bits():
    """x, y and dx of more than 2^31 elements, and weights' gradients that sum over all rows."""
    n, d, f = 2100000, 1024, 64
    x = big(n, d)
    ws = [(rn(gen(i), *s) * s[1] ** -0.5).bfloat16() for i, s in enumerate(((f, d), (f, d), (d, f)))]
    last = slice(n - 400, n)

    def run(x):
        leaf = x.detach().requires_grad_(True)
        y = ops.gated_ffn(leaf, *ws)
        return y.detach(), torch.autograd.grad(y, leaf, x)[0]

    # products are split over k by a rule on the sizes; at k = 64 and 128 neither call splits, so the bits are equal
    for a, b in zip(run(x), run(x[last])):
        assert torch.equal(a[last], b)
    assert ops.status() == 0
