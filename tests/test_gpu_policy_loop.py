"""The policy operators together, as examples/policy_loop.py runs them on NetModule's observations."""
import importlib
import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ib = importlib.import_module("isaac-net_b200")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("policy_loop", os.path.join(ROOT, "examples", "policy_loop.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_the_example_runs_and_repeats():
    ex = example()
    a = ex.main(envs=8, robots=16, steps=4, verbose=False)
    b = ex.main(envs=8, robots=16, steps=4, verbose=False)
    assert a == b and all(x == x for row in a for x in row)      # no operator depends on the order that blocks run in
    assert a[0][1] > 0.0


def logits64(p, obs, keep=None):
    """The policy of the example in 64 bits, rounding to bf16 where it does; keep: dropout masks with their scale."""
    r = lambda t: t.bfloat16().double()
    w = lambda t: t.detach().double()
    rms = lambda v: v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    x = r(obs.double().bfloat16().double() @ w(p.embed).T)
    cond = r(x.mean(1, keepdim=True))
    n = r(rms(x) * w(p.first))
    for i, b in enumerate(p.blocks):
        g = n @ w(b["w_gate"]).T
        h = r(r(g * torch.sigmoid(g) * (n @ w(b["w_up"]).T)) @ w(b["w_down"]).T)
        if keep is not None:
            h = r(h * keep[i])
        gate = r(torch.sigmoid(r(cond @ w(b["gate"]).T)))
        y = x + 0.5 * gate * (w(b["post"]) * rms(h))
        x, n = r(y), r(rms(y) * w(b["next"]))
    return r(n @ w(p.head).T)


@pytest.mark.parametrize("envs,robots", [(1, 1), (5, 3), (64, 16)])
def test_policy_logits_against_64_bits(envs, robots):
    """bf16 activations of a 2-block net: each of its about 12 roundings moves a logit by at most 2^-8 of the activations'
    size, and a random walk of them by about 4 times that."""
    ex = example()
    ops = ib.policy_ops
    p = ex.Policy(11, 5, D=128, F=200)
    g = torch.Generator(device="cuda").manual_seed(2)
    obs = torch.randn(envs, robots, 11, generator=g, device="cuda")
    with torch.no_grad():
        got = p.logits(obs).double()
    want = logits64(p, obs)
    assert float((got - want).norm() / want.norm()) < 12 * 2.0 ** -8
    # with dropout: the mask from a call on ones
    env = torch.arange(envs, device="cuda") + 40
    key = (eng_mod.seed_key(3), env, torch.zeros_like(env), torch.full_like(env, 9))
    ones = torch.ones(envs, robots, 128, dtype=torch.bfloat16, device="cuda")
    keep = [ops.counter_dropout(ones, ex.P_DROP, *key, stream=i).double() for i in range(2)]
    with torch.no_grad():
        got = p.logits(obs, drop=key).double()
    want = logits64(p, obs, keep)
    assert float((got - want).norm() / want.norm()) < 12 * 2.0 ** -8


def test_actions_do_not_depend_on_the_split():
    """Half of the envs, with their global ids, act as they do in the whole batch (same dropout, same draws)."""
    ex = example()
    ops = ib.policy_ops
    p = ex.Policy(9, 4, D=64, F=96)
    g = torch.Generator(device="cuda").manual_seed(4)
    obs = torch.randn(12, 16, 9, generator=g, device="cuda")
    env = torch.arange(12, device="cuda")
    ep, ctr = env % 3, env * 7

    def run(sl):
        with torch.no_grad():
            logits = p.logits(obs[sl], drop=(77, env[sl], ep[sl], ctr[sl]))
            u = ops.uniforms(77, 16, env[sl], ep[sl], ctr[sl], stream=1)
            return ops.sample_logits(logits, u, temperature=0.9)

    whole = run(slice(0, 12))
    for sl in (slice(0, 5), slice(5, 12)):
        tok, logp = run(sl)
        assert torch.equal(tok, whole[0][sl]) and torch.equal(logp, whole[1][sl])


def test_uniforms_are_the_engines_draws():
    """uniforms() against the host hash of the counter RNG: element i of an env is mix(mix(key + i GOLD) ^ key) >> 8, 24 bits."""
    ops = ib.policy_ops
    mix, salt = eng_mod._mix32, eng_mod._salt
    env, ep, ctr = torch.tensor([5, 2 ** 33 + 1]), torch.tensor([0, 3]), torch.tensor([7, 0])
    got = ops.uniforms(99, 6, env.cuda(), ep.cuda(), ctr.cuda(), stream=4).cpu()
    for e in range(2):
        k = mix(99 ^ salt(int(env[e])))
        for v in (int(ep[e]), 0x53, int(ctr[e]), 4):
            k = mix(k ^ salt(v))
        for i in range(6):
            h = mix(mix((k + i * 0x9E3779B9) & 0xFFFFFFFF) ^ k)
            assert float(got[e, i]) == (h >> 8) * 2.0 ** -24
    with pytest.raises(ValueError):
        ops.uniforms(99, 6, env)


def test_policy_in_a_cuda_graph():
    """A captured forward pass replays to the eager pass's bits."""
    ex = example()
    p = ex.Policy(8, 4, D=128, F=256)
    obs = torch.randn(32, 16, 8, device="cuda")
    with torch.no_grad():
        want = p.logits(obs)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            p.logits(obs)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = p.logits(obs)
        g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
