"""A policy in the loop of the simulated network: NetModule's observations through residual blocks of the policy operators,
a message class for every robot drawn from its logits, the answer sent back as a TrafficRequest, and a policy gradient step.

    python examples/policy_loop.py [--envs 64] [--robots 16] [--steps 20]

One residual block is block_norm (post-norm, gate, residual scale and the next block's pre-norm in one pass) around
gated_ffn and counter_dropout; sample_logits draws the classes from uniforms of the engine's counter RNG.  Everything that
is random is keyed by the global env id, so a batch split over several engines acts as the whole one does.
"""
import argparse
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
ib = importlib.import_module("isaac-net_b200")
presets = importlib.import_module("isaac-net_b200.presets")
ops = ib.policy_ops

P_DROP, SCALE, STREAM_ACT = 0.1, 0.5, 100


class Policy:
    """obs [E, R, dim] -> logits [E, R, classes].  Blocks of width D with hidden width F, bf16; each env has a gate per
    block, made from its robots' mean embedding."""

    def __init__(self, dim, classes, D=256, F=704, blocks=2, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s, std: (torch.randn(*s, generator=g) * std).to(device, torch.bfloat16).requires_grad_(True)
        one = lambda *s: torch.ones(*s, dtype=torch.bfloat16, device=device, requires_grad=True)
        self.embed, self.head = mk(D, dim, std=dim ** -0.5), mk(classes, D, std=0.1 * D ** -0.5)
        self.first = one(D)
        self.blocks = [dict(gate=mk(D, D, std=D ** -0.5), w_gate=mk(F, D, std=D ** -0.5), w_up=mk(F, D, std=D ** -0.5),
                            w_down=mk(D, F, std=F ** -0.5), post=one(D), next=one(D)) for _ in range(blocks)]

    def parameters(self):
        return [self.embed, self.head, self.first, *(p for b in self.blocks for p in b.values())]

    def logits(self, obs, drop=None):
        """drop: None, or the key of this step's dropout (s0, env_id, episode, ctr)."""
        x = obs.to(torch.bfloat16) @ self.embed.T
        cond = x.mean(1, keepdim=True)                          # [E, 1, D]
        n = ops.block_norm(x, self.first)
        for i, b in enumerate(self.blocks):
            h = ops.gated_ffn(n, b["w_gate"], b["w_up"], b["w_down"])
            if drop is not None:
                h = ops.counter_dropout(h, P_DROP, *drop, stream=i)
            gate = torch.sigmoid(cond @ b["gate"].T)
            x, n = ops.block_norm(x, b["next"], h, post_weight=b["post"], gate=gate, scale=SCALE)
        return (n @ self.head.T).float()


def step_key(net):
    """What this step's dropout is keyed by; copies, because the engine's counters move on in place."""
    return net.eng.s0, net.eng.env_id, net.eng.episode.clone(), net.clock.clone()


def act(policy, net, obs, drop=None):
    """The message class of every robot this step: (send [E, R], its log-probability).  Drawn from all classes: a filter
    (top-k, top-p, min-p) would make logp that of another distribution than log_prob's."""
    eng = net.eng
    with torch.no_grad():
        logits = policy.logits(obs, drop)
        u = ops.uniforms(eng.s0, net.R, eng.env_id, eng.episode, net.clock, stream=STREAM_ACT)
        return ops.sample_logits(logits, u)


def log_prob(policy, obs, send, drop=None):
    """The log-probability of the classes `send`, with its gradient; drop: that of the call of act that drew them."""
    return torch.log_softmax(policy.logits(obs, drop), -1).gather(-1, send[..., None])[..., 0]


def main(envs=64, robots=16, steps=20, lr=0.05, verbose=True):
    wl = presets.workload(1)
    cfg = wl.config(traffic=(), msg_sizes=(200.0, 1500.0, 8192.0))
    net = ib.NetModule("L2", envs, robots, "cuda", cfg, seed=wl.seed, isaac=ib.IsaacNetCfg(
        radio="engine", obs_features=("aoi", "sinr", "queue_len", "last_delivered", "delay_history")))
    motion = presets.Motion(1, envs, robots, seed=wl.seed)
    policy = Policy(net.obs_dim, classes=1 + len(cfg.msg_sizes))     # class 0: send nothing
    net.reset()
    pos, log = motion.current(), []
    for step in range(steps):
        obs = net.obs()
        key = step_key(net)
        send, logp = act(policy, net, obs, key)
        net.submit(None, ib.TrafficRequest(send))
        out = net.step(None, pos.cuda())
        pos = motion.advance()
        # one policy gradient step: fresh information, few queued bytes
        reward = -out["aoi_s"] - 1e-6 * out["queue_bytes"]
        adv = (reward - reward.mean()) / (reward.std() + 1e-6)
        loss = -(adv * log_prob(policy, obs, send, key)).mean()
        for p, g in zip(policy.parameters(), torch.autograd.grad(loss, policy.parameters())):
            with torch.no_grad():
                p -= lr * g
        log.append((float(loss.detach()), float(out["aoi_s"].mean()), float(logp.mean())))
        if verbose:
            print(f"step {step:3d}  loss {log[-1][0]:+.4f}  mean AoI {log[-1][1] * 1e3:6.1f} ms  mean logp {log[-1][2]:+.3f}")
    return log


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("envs", 64), ("robots", 16), ("steps", 20)):
        ap.add_argument("--" + name, type=int, default=value)
    main(**vars(ap.parse_args()))
