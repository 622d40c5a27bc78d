"""The policy's memory and distill_loss where calls go beyond the plain ones: refusals, layouts, resets against what an episode
left behind, graphs, streams, long tensors, and a run of them together on the simulated network.  Tolerances as in the
operators' own test files."""
import importlib
import math
import os
import sys

import pytest
import torch

ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DT = [torch.bfloat16, torch.float16, torch.float32]
Unsupported = eng_mod.B200Unsupported


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rn(g, *s):
    return torch.randn(*s, generator=g, device="cuda")


def scan_args(g, e, r, t, ch, n, dtype):
    mk = lambda *s: rn(g, e, r, t, *s).to(dtype)
    return dict(x=mk(ch), dt=mk(ch), a=-torch.rand(ch, n, generator=g, device="cuda"), b=mk(n), c=mk(n)), \
        dict(d=rn(g, ch), z=mk(ch), dt_bias=rn(g, ch) - 1, state=rn(g, e, r, ch, n))


def test_refusals():
    g = gen(0)
    x, w, b = rn(g, 2, 3, 5, 8), rn(g, 8, 4), rn(g, 8)
    st = rn(g, 2, 3, 3, 8)
    flag = torch.zeros(2, 1, 5, dtype=torch.bool, device="cuda")
    for kind, f in [
            (Unsupported, lambda: ops.causal_conv(x.double(), w, b)), (Unsupported, lambda: ops.causal_conv(x, w[:, :1], b)),
            (Unsupported, lambda: ops.causal_conv(x, rn(g, 8, 5))), (TypeError, lambda: ops.causal_conv(x, w.half())),
            (TypeError, lambda: ops.causal_conv(x, w, b.bfloat16())), (Unsupported, lambda: ops.causal_conv(x, w.cpu())),
            (ValueError, lambda: ops.causal_conv(x, w[:7])), (ValueError, lambda: ops.causal_conv(x, w, b[:7])),
            (ValueError, lambda: ops.causal_conv(x[0, 0, 0], w)), (ValueError, lambda: ops.causal_conv(x, w, state=st[:, :, :2])),
            (TypeError, lambda: ops.causal_conv(x, w, state=st.half())), (ValueError, lambda: ops.causal_conv(x, w, act="gelu")),
            (TypeError, lambda: ops.causal_conv(x, w, reset=flag.float())), (ValueError, lambda: ops.causal_conv(x, w, reset=flag[..., :4])),
            (ValueError, lambda: ops.causal_conv(x, w, reset=flag[:1].expand(1, 3, 5))),
            (ValueError, lambda: ops.causal_conv(x, w, reset=flag[0].expand(3, 5))),      # a flag per robot, for no env
            (TypeError, lambda: ops.causal_conv(x, None)),
            (ValueError, lambda: ops.causal_conv_step(x[:, :, 0], w, st[..., :1].expand(2, 3, 3, 8))),
            (ValueError, lambda: ops.causal_conv_step(x[:, :, 0], w, st[:1, :1].expand(2, 3, 3, 8))),
            (ValueError, lambda: ops.causal_conv_step(x[:, :, 0], w, st.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3))),
            (Unsupported, lambda: ops.causal_conv_step(x[:, :, 0], w.clone().requires_grad_(True), st))]:
        with pytest.raises(kind):
            f()
    p, q = scan_args(g, 2, 3, 5, 8, 4, torch.float32)
    call = lambda **kw: ops.selective_scan(**{**p, **q, **kw})
    for kind, kw in [(Unsupported, dict(x=p["x"].double())), (TypeError, dict(dt=p["dt"].half())), (ValueError, dict(dt=p["dt"][..., :7])),
                     (TypeError, dict(a=p["a"].half())), (ValueError, dict(a=p["a"][:7])), (ValueError, dict(a=p["a"][0])),
                     (ValueError, dict(b=p["b"][..., :3])), (ValueError, dict(c=p["c"][:, :, :4])), (TypeError, dict(c=p["c"].half())),
                     (ValueError, dict(d=q["d"][:7])), (TypeError, dict(d=q["d"].half())), (ValueError, dict(z=q["z"][:1])),
                     (ValueError, dict(dt_bias=q["dt_bias"][:3])), (ValueError, dict(state=q["state"][:1])),
                     (TypeError, dict(state=q["state"].half())), (Unsupported, dict(x=p["x"].cpu())), (Unsupported, dict(z=q["z"].cpu())),
                     (Unsupported, dict(a=-torch.ones(8, 65, device="cuda"))), (TypeError, dict(reset=flag.int())),
                     (ValueError, dict(reset=flag[:, :, :3]))]:
        with pytest.raises(kind):
            call(**kw)
    one = {k: v[:, :, 0] if k in ("x", "dt", "b", "c", "z") else v for k, v in {**p, **q}.items()}
    with pytest.raises(Unsupported):
        ops.selective_scan_step(**{**one, "a": one["a"].clone().requires_grad_(True)})
    with pytest.raises(ValueError):
        ops.selective_scan_step(**{**one, "state": one["state"].transpose(-1, -2).contiguous().transpose(-1, -2)})
    l, t, i = rn(g, 4, 9), rn(g, 4, 3), torch.zeros(4, 3, dtype=torch.long, device="cuda")
    for kind, f in [(ValueError, lambda: ops.distill_loss(l, t[:3], i)), (ValueError, lambda: ops.distill_loss(l, t, i[:, :2])),
                    (TypeError, lambda: ops.distill_loss(l, t, i.int())), (ValueError, lambda: ops.distill_loss(l, t, i, temperature=0.0)),
                    (ValueError, lambda: ops.distill_loss(l, t, i, temperature=math.nan)), (Unsupported, lambda: ops.distill_loss(l.double(), t, i)),
                    (Unsupported, lambda: ops.distill_loss(l, t.double(), i)), (Unsupported, lambda: ops.distill_loss(l, t.cpu(), i)),
                    (ValueError, lambda: ops.distill_loss(l, t, i, mask=torch.ones(4, 8, dtype=torch.bool, device="cuda"))),
                    (TypeError, lambda: ops.distill_loss(l, t, i, mask=torch.ones(4, 9, device="cuda"))),
                    (Unsupported, lambda: ops.distill_loss(l, t.clone().requires_grad_(True), i)),
                    (Unsupported, lambda: ops.distill_loss(l, rn(g, 4, 1025), torch.zeros(4, 1025, dtype=torch.long, device="cuda")))]:
        with pytest.raises(kind):
            f()


def test_derivatives_of_derivatives_and_tangents_are_refused():
    g = gen(1)
    p, q = scan_args(g, 1, 2, 6, 8, 4, torch.float32)
    x = p["x"].requires_grad_(True)
    for f in (lambda: ops.selective_scan(**p, **q)[0], lambda: ops.causal_conv(x, rn(g, 8, 4))[0],
              lambda: ops.distill_loss(x, x.detach()[..., :2], torch.zeros(1, 2, 6, 2, dtype=torch.long, device="cuda"))):
        gx, = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(gx.sum(), x)
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        dual = fw.make_dual(x.detach(), torch.ones_like(x))
        for f in (lambda: ops.causal_conv(dual, rn(g, 8, 4)), lambda: ops.selective_scan(dual, *list(p.values())[1:]),
                  lambda: ops.distill_loss(dual, x.detach()[..., :2], torch.zeros(1, 2, 6, 2, dtype=torch.long, device="cuda"))):
            with pytest.raises(Unsupported):
                f()


def test_empty_batches_and_no_steps():
    g = gen(2)
    w = rn(g, 8, 3)
    for shape in ((0, 3, 5, 8), (2, 0, 5, 8), (2, 3, 0, 8)):
        x = torch.zeros(*shape, device="cuda").requires_grad_(True)
        st = rn(g, *shape[:2], 2, 8).requires_grad_(True)
        wl = w.clone().requires_grad_(True)
        y, new = ops.causal_conv(x, wl, state=st)
        assert y.shape == x.shape and torch.equal(new, st)
        gx, gw, gs = torch.autograd.grad((y, new), (x, wl, st), (torch.ones_like(y), torch.full_like(new, 2.0)))
        assert bool((gw == 0).all()) and bool((gs == 2).all())
        h = rn(g, *shape[:2], 8, 4).requires_grad_(True)
        bc = torch.zeros(*shape[:3], 4, device="cuda")
        a = -torch.ones(8, 4, device="cuda").requires_grad_(True)
        y, new = ops.selective_scan(x, x.detach(), a, bc, bc, state=h)
        assert y.shape == x.shape and torch.equal(new, h)
        ga, gh = torch.autograd.grad((y, new), (a, h), (torch.ones_like(y), torch.full_like(new, 3.0)), allow_unused=True)
        assert bool((gh == 3).all())
        assert bool((ops.causal_conv(x.detach(), w)[1] == 0).all())
    l = torch.zeros(0, 7, device="cuda").requires_grad_(True)
    loss = ops.distill_loss(l, l.detach()[:, :2], torch.zeros(0, 2, dtype=torch.long, device="cuda"))
    assert loss.shape == (0,) and torch.autograd.grad(loss.sum(), l)[0].shape == l.shape


@pytest.mark.parametrize("dtype", DT)
def test_nothing_of_an_ended_episode_is_seen(dtype):
    """NaN and infinities before a reset leave the episode after it with the values of a run that begins there, forward and
    backward; the convolution's with its bits.  The scan's steps lie elsewhere in their chunks of eight, at whose ends a state is
    raised by up to 3.2 * 2^-24, so both runs are within the bound of test_gpu_policy_memory.py of the true value: with 12
    steps, delta a below 3 and |v| below 5 it is 2 * 12 * (4 + 3 * 31 + 2) u = 2400 u = 1.4e-4 of the largest, and a rounding."""
    near = lambda p, q: bool(((p.double() - q.double()).abs() <= torch.finfo(p.dtype).eps * q.double().abs() + 2.8e-4 * q.double().abs().max()).all())
    g = gen(3)
    t, cut = 21, 9
    p, q = scan_args(g, 2, 3, t, 40, 16, dtype)
    w, b = rn(g, 40, 4).to(dtype), rn(g, 40).to(dtype)
    flags = torch.zeros(2, 1, t, dtype=torch.bool, device="cuda")
    flags[..., cut] = True
    seqs = ("x", "dt", "b", "c")
    bad = {k: v.clone() for k, v in p.items()}
    bad["x"][:, :, 3, 5] = math.nan
    bad["x"][:, :, cut - 1, 6] = math.inf
    z = q["z"].clone()
    gy = rn(g, 2, 3, t, 40).to(dtype)
    gy[:, :, :cut] = 0
    late = lambda v: v[:, :, cut:].contiguous()

    def run(args, z, state, reset, gy):
        leaf = {k: args[k].detach().clone().requires_grad_(True) for k in ("x", "dt", "b", "c")}
        y, new = ops.selective_scan(leaf["x"], leaf["dt"], args["a"], leaf["b"], leaf["c"], d=q["d"], z=z, dt_bias=q["dt_bias"],
                                    state=state, reset=reset)
        v, last = ops.causal_conv(leaf["x"], w, b, reset=reset)
        gs = torch.autograd.grad((y, v), list(leaf.values()), (gy, gy))
        return y.detach(), new.detach(), v.detach(), last.detach(), gs

    one = run(bad, z, q["state"].clone().fill_(math.inf), flags, gy)
    two = run({k: late(v) if k in seqs else v for k, v in p.items()}, late(z), None, None, late(gy))
    assert near(one[1], two[1]) and torch.equal(one[3], two[3])
    assert near(one[0][:, :, cut:], two[0]) and torch.equal(one[2][:, :, cut:], two[2])
    for a, c in zip(one[4], two[4]):
        assert near(a[:, :, cut:], c)


@pytest.mark.parametrize("dtype", DT)
def test_steps_of_no_length_leave_the_state(dtype):
    """dt of -inf or of the type's lowest value: delta is 0, the state stays as it was to the bit, no gradient is NaN; very large
    dt forget everything; a NaN is not hidden."""
    g = gen(12)
    p, q = scan_args(g, 2, 2, 12, 40, 16, dtype)
    x, w = p["x"], [3, 4, 9]
    for low in (-math.inf, torch.finfo(dtype).min):
        dt = p["dt"].clone()
        dt[:, :, w] = low
        leaf = {k: v.detach().clone().requires_grad_(True) for k, v in {**p, "dt": dt, **q}.items()}
        y, new = ops.selective_scan(**leaf)
        grads = torch.autograd.grad((y.float().sum() + new.sum()), list(leaf.values()))
        assert all(bool(v.isfinite().all()) for v in (y, new, *grads))
        assert bool((grads[1][:, :, w] == 0).all())
        one = {k: v[:, :, 3] if k in ("x", "dt", "b", "c", "z") else v for k, v in {**p, "dt": dt, **q}.items()}
        st = q["state"].clone()
        ops.selective_scan_step(**{**one, "state": st})
        assert torch.equal(st, q["state"])
    dt = p["dt"].clone()
    dt[:, :, 11] = 1e4
    y, new = ops.selective_scan(**{**p, "dt": dt, "a": p["a"] - 1}, **q)
    v = dt[:, :, 11].float() + q["dt_bias"]
    want = (v * x[:, :, 11].float())[..., None] * p["b"][:, :, 11, None].float()
    assert torch.allclose(new, want, rtol=1e-6, atol=1e-3)
    dt[0, 0, 5, 7] = math.nan
    y, new = ops.selective_scan(**{**p, "dt": dt, "a": p["a"] - 1}, **q)
    assert bool(y[0, 0, 5:, 7].isnan().all()) and bool(new[0, 0, 7].isnan().all()) and int(new.isnan().sum()) == 16


def test_layouts_and_strides():
    """Views of wider buffers, rows that start anywhere, expanded inputs and gradients, transposed envs: the values of the
    contiguous call, to the bit where its form is the same."""
    g = gen(4)
    for dtype in DT:
        wide = rn(g, 3, 4, 9, 70).to(dtype)
        w, b = rn(g, 64, 4).to(dtype), rn(g, 64).to(dtype)
        want, last = ops.causal_conv(wide[..., :64].contiguous(), w, b)
        for x in (wide[..., :64], wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :64],
                  wide[..., :64].contiguous().flip(0).flip(0)):
            y, s = ops.causal_conv(x, w, b)
            assert torch.equal(y, want) and torch.equal(s, last)
        off = wide[..., 3:67]
        assert torch.equal(ops.causal_conv(off, w, b)[0], ops.causal_conv(off.contiguous(), w, b)[0])
        x = rn(g, 1, 1, 9, 64).to(dtype).expand(3, 4, 9, 64).detach().requires_grad_(True)
        y, s = ops.causal_conv(x, w, b)
        gx, = torch.autograd.grad(y.sum(), x)                     # an expanded gradient
        gy = torch.ones(3, 4, 9, 64, dtype=dtype, device="cuda")
        x2 = x.detach().contiguous().requires_grad_(True)
        assert torch.equal(gx, torch.autograd.grad(ops.causal_conv(x2, w, b)[0], x2, gy)[0])
        p, q = scan_args(g, 3, 4, 9, 64, 16, dtype)
        want, last = ops.selective_scan(**p, **q)
        bc = torch.cat((p["b"], p["c"]), -1)
        y, s = ops.selective_scan(**{**p, "b": bc[..., :16], "c": bc[..., 16:]}, **q)
        assert torch.equal(y, want) and torch.equal(s, last)
        tm = lambda v: v.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
        y, s = ops.selective_scan(tm(p["x"]), tm(p["dt"]), p["a"], tm(p["b"]), tm(p["c"]), **{**q, "z": tm(q["z"])})
        assert torch.equal(y, want) and torch.equal(s, last) and y.stride() == tm(p["x"]).stride()
        y, s = ops.selective_scan(**{**p, "dt": p["dt"][..., :1].expand_as(p["dt"])}, **q)       # one step length a robot
        y2, s2 = ops.selective_scan(**{**p, "dt": p["dt"][..., :1].expand_as(p["dt"]).contiguous()}, **q)
        assert torch.equal(y, y2) and torch.equal(s, s2)


def test_steps_write_their_states_and_nothing_else():
    """States that are views of a wider buffer, a batch of which some robots start an episode, and what lies between.  A state
    off 16 bytes is another form's, whose sum of N products <h, c> has another order: each is N u off its terms' absolute sum."""
    g = gen(5)
    for dtype in DT:
        for c, k, n in ((24, 4, 16), (33, 2, 5)):
            pool = rn(g, 5, (k - 1) * c + 7).to(dtype)
            before = pool.clone()
            st = pool[:, :(k - 1) * c].view(5, k - 1, c)
            x, w = rn(g, 5, c).to(dtype), rn(g, c, k).to(dtype)
            reset = torch.tensor([False, True, False, False, True], device="cuda")
            y = ops.causal_conv_step(x, w, st, reset=reset)
            want, new = ops.causal_conv(x[:, None], w, state=before[:, :(k - 1) * c].reshape(5, k - 1, c), reset=reset[:, None])
            assert torch.equal(y, want[:, 0]) and torch.equal(st, new) and torch.equal(pool[:, (k - 1) * c:], before[:, (k - 1) * c:])
            pool = rn(g, 5, c * n + 3)
            before = pool.clone()
            st = pool[:, :c * n].view(5, c, n)
            p, q = scan_args(g, 5, 1, 1, c, n, dtype)
            one = {k2: v[:, 0, 0] if k2 in ("x", "dt", "b", "c", "z") else v for k2, v in {**p, **q}.items()}
            y = ops.selective_scan_step(**{**one, "state": st}, reset=reset)
            clean = before[:, :c * n].reshape(5, c, n).clone()
            y2 = ops.selective_scan_step(**{**one, "state": clean}, reset=reset)
            assert torch.equal(st, clean) and torch.equal(pool[:, c * n:], before[:, c * n:])
            z = one["z"].double()
            mag = ((clean.double().abs() * one["c"].double().abs()[:, None]).sum(-1) + (q["d"] * one["x"]).double().abs()) * (z * torch.sigmoid(z)).abs()
            assert bool(((y.double() - y2.double()).abs() <= torch.finfo(dtype).eps * y2.double().abs() + (2 * n + 4) * 2.0 ** -24 * mag).all())


def test_a_step_in_place_is_seen_by_autograd():
    g = gen(6)
    p, q = scan_args(g, 2, 3, 5, 16, 8, torch.float32)
    leaf = p["x"].requires_grad_(True)
    y, _ = ops.selective_scan(**p, **q)
    with torch.no_grad():
        one = {k: v[:, :, 0] if k in ("x", "dt", "b", "c", "z") else v for k, v in {**p, **q}.items()}
        ops.selective_scan_step(**one)                              # updates the state that the backward pass needs
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), leaf)
    x, w, st = rn(g, 2, 5, 16).requires_grad_(True), rn(g, 16, 4), rn(g, 2, 3, 16)
    y, _ = ops.causal_conv(x, w, state=st)
    with torch.no_grad():
        ops.causal_conv_step(x[:, 0], w, st)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)
    with torch.inference_mode():
        s = torch.zeros(2, 3, 16, device="cuda")
        ops.causal_conv_step(x.detach()[:, 0], w, s)


def test_repeated_calls_have_equal_bits():
    g = gen(7)
    for e, r, t, ch, n in ((64, 16, 16, 130, 16), (1, 1, 2000, 100, 10)):
        p, q = scan_args(g, e, r, t, ch, n, torch.bfloat16)
        leaf = {k: v.requires_grad_(True) for k, v in {**p, **q}.items()}
        gy = rn(g, e, r, t, ch).bfloat16()
        w = rn(g, ch, 4).bfloat16().requires_grad_(True)
        first = None
        for _ in range(4):
            y, new = ops.selective_scan(**leaf)
            v, _ = ops.causal_conv(leaf["x"], w)
            got = [y, new, v, *torch.autograd.grad((y, v), [*leaf.values(), w], (gy, gy))]
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(got, first))
    logits = rn(g, 300, 5001)
    i = torch.randint(0, 5001, (300, 40), generator=g, device="cuda")
    l = logits.requires_grad_(True)
    got = [torch.autograd.grad(ops.distill_loss(l, i.float() * 1e-3, i).sum(), l)[0] for _ in range(3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_graphs_replay_a_control_loop_and_a_training_step():
    """A captured control step whose states live on from replay to replay, and a captured training step, against the same
    calls made one by one; two graphs that share nothing are replayed in turn."""
    g = gen(8)
    c, n = 64, 16
    w, b = rn(g, c, 4).bfloat16(), rn(g, c).bfloat16()
    p, q = scan_args(g, 4, 3, 1, c, n, torch.bfloat16)
    one = {k: v[:, :, 0].contiguous() if k in ("x", "dt", "b", "c", "z") else v for k, v in {**p, **q}.items()}
    reset = torch.zeros(4, 1, dtype=torch.bool, device="cuda")
    cs = rn(g, 4, 3, 3, c).bfloat16()
    x = rn(g, 4, 3, c).bfloat16()

    def act(x, cs, hs):
        v = ops.causal_conv_step(x, w, cs, b, reset=reset)
        return ops.selective_scan_step(**{**one, "x": v, "state": hs}, reset=reset)

    tx = rn(g, 4, 3, 70, c).bfloat16()
    tp, tq = scan_args(g, 4, 3, 70, c, n, torch.bfloat16)
    leaf = [t.clone().requires_grad_(True) for t in (tx, w, b, tp["a"])]
    ti = torch.randint(0, c, (4, 3, 70, 5), generator=g, device="cuda")

    def train(leaf):
        v, _ = ops.causal_conv(leaf[0], leaf[1], leaf[2])
        y, _ = ops.selective_scan(v, tp["dt"], leaf[3], tp["b"], tp["c"], **tq)
        loss = ops.distill_loss(y, tp["x"][..., :5], ti)
        return [loss.detach(), *torch.autograd.grad(loss.sum(), leaf)]

    live = [cs.clone(), one["state"].clone()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        act(x, cs.clone(), one["state"].clone())
        train([t.detach().clone().requires_grad_(True) for t in leaf])
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        out = act(x, *live)
    with torch.cuda.graph(g2):
        got = train(leaf)
    for t, s in zip(live, (cs, one["state"])):
        t.copy_(s)
    eager = [cs.clone(), one["state"].clone()]
    for k in range(4):
        x.copy_(rn(g, 4, 3, c))
        reset.copy_(torch.rand(4, 1, generator=g, device="cuda") < 0.3)
        with torch.no_grad():
            leaf[0].copy_(rn(g, 4, 3, 70, c))
        g1.replay()
        g2.replay()
        want = act(x, *eager)
        assert torch.equal(out, want) and all(torch.equal(a, e) for a, e in zip(live, eager))
        ref = train([t.detach().clone().requires_grad_(True) for t in leaf])
        assert all(torch.equal(a, e) for a, e in zip(got, ref))


def test_other_streams():
    """Calls on streams of their own, two at once: the bits of the calls on the default stream."""
    g = gen(9)
    p, q = scan_args(g, 8, 4, 40, 96, 16, torch.float16)
    leaf = {k: v.requires_grad_(True) for k, v in {**p, **q}.items()}
    w = rn(g, 96, 3).half().requires_grad_(True)
    gy = rn(g, 8, 4, 40, 96).half()

    def run():
        v, _ = ops.causal_conv(leaf["x"], w)
        y, _ = ops.selective_scan(**{**leaf, "x": v})
        return [y.detach(), *torch.autograd.grad(y, [*leaf.values(), w], gy)]

    want = run()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


def test_tensors_of_more_than_2_31_elements():
    """The last sequences of a batch whose offsets pass 32 bits have the bits of a call on them alone."""
    g = gen(10)
    s, t, c = 131100, 16, 1030                              # 2.16e9 elements; rows of 1030: not aligned to 16 bytes
    x = torch.empty(s, t, c, dtype=torch.bfloat16, device="cuda")
    for k in range(0, s, 8192):
        x[k:k + 8192] = torch.randn(x[k:k + 8192].shape, generator=g, device="cuda", dtype=torch.bfloat16)
    w, b = rn(g, c, 4).bfloat16(), rn(g, c).bfloat16()
    last = slice(s - 3, s)
    y, new = ops.causal_conv(x, w, b)
    y1, new1 = ops.causal_conv(x[last].clone(), w, b)
    assert torch.equal(y[last], y1) and torch.equal(new[last], new1)
    leaf, small = x.requires_grad_(True), x.detach()[last].clone().requires_grad_(True)
    gx, = torch.autograd.grad(ops.causal_conv(leaf, w, b)[0], leaf, y)
    g1, = torch.autograd.grad(ops.causal_conv(small, w, b)[0], small, y1)
    assert torch.equal(gx[last], g1)
    del gx, y, new
    x = x.detach()
    bc = rn(g, s, t, 4).bfloat16()
    a = -torch.rand(c, 4, generator=g, device="cuda")
    y, new = ops.selective_scan(x, x, a, bc, bc)
    y1, new1 = ops.selective_scan(x[last].clone(), x[last].clone(), a, bc[last].clone(), bc[last].clone())
    assert torch.equal(y[last], y1) and torch.equal(new[last], new1)
    del x, y, new
    rows, v = 66000, 32769
    l = torch.empty(rows, v, dtype=torch.bfloat16, device="cuda")
    for k in range(0, rows, 4096):
        l[k:k + 4096] = torch.randn(l[k:k + 4096].shape, generator=g, device="cuda", dtype=torch.bfloat16)
    i = torch.randint(0, v, (rows, 6), generator=g, device="cuda")
    i[-1, -1] = v - 1
    tl = rn(g, rows, 6)
    l = l.requires_grad_(True)
    loss = ops.distill_loss(l, tl, i)
    gl, = torch.autograd.grad(loss.sum(), l)
    tail = l.detach()[-5:].requires_grad_(True)              # a view: its rows start where they did
    loss1 = ops.distill_loss(tail, tl[-5:], i[-5:])
    g1, = torch.autograd.grad(loss1.sum(), tail)
    assert torch.allclose(loss[-5:], loss1, rtol=1e-5, atol=1.5e-5)
    # one step of bf16, and q and p to 1.5e-5
    assert bool(((gl[-5:].float() - g1.float()).abs() <= 2.0 ** -7 * g1.float().abs() + 1.5e-5).all())


def test_memory_policy_rollout_equals_its_steps():
    """The example's policy: logits of a rollout with resets against those of its steps.  Both round to bf16 at the same places,
    but the scan's sums have another order, so that its outputs, the product after it and their sum may each round apart by
    a step of 2^-8: within 2^-6 of the largest logit."""
    sys.path.insert(0, ROOT)
    ex = importlib.import_module("examples.policy_memory") if os.path.isdir(os.path.join(ROOT, "examples")) else None
    g = gen(11)
    pol = ex.MemoryPolicy(12, 7, D=64)
    obs = rn(g, 3, 5, 14, 12)
    reset = torch.rand(3, 1, 14, generator=g, device="cuda") < 0.2
    memory = pol.start(3, 5)
    logits, after = pol.rollout(obs, reset, [m.clone() for m in memory])
    plain = logits.detach()
    for t in range(14):
        one = pol.step(obs[:, :, t], reset[..., t], memory)
        assert float((one - plain[:, :, t]).abs().max()) <= 2.0 ** -6 * float(plain.abs().max())
    assert torch.equal(memory[0], after[0])
    grads = torch.autograd.grad(logits.square().mean(), pol.parameters())
    assert all(bool(q.isfinite().all()) and float(q.abs().max()) > 0 for q in grads)


def test_memory_example_runs():
    sys.path.insert(0, ROOT)
    ex = importlib.import_module("examples.policy_memory")
    log = ex.main(envs=8, robots=4, rollouts=2, length=6, verbose=False)
    assert len(log) == 2 and all(math.isfinite(v) for v in log)
