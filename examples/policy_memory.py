"""A policy with a memory, distilled from a teacher's logged answers on the simulated network: the robots act step by step
through the memory's one-step forms, every few control steps the rollout is replayed as a whole, with the envs' resets
inside, and the student is trained on the teacher's top logits.

    python examples/policy_memory.py [--envs 64] [--robots 16] [--rollouts 4] [--length 16]

The memory is one residual block: block_norm, a projection, causal_conv, selective_scan (whose steps, b and c come from a second
projection), a projection back.  The teacher sees what the student must remember: the observations of the last steps.
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

TAPS, STATES, RANK, TOP = 4, 16, 16, 4


class MemoryPolicy:
    """obs [..., dim] -> logits [..., classes], with a memory of width D per robot; bf16, the memory's parameters fp32."""

    def __init__(self, dim, classes, D=128, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)
        mk = lambda *s, std: (torch.randn(*s, generator=g) * std).to(device, torch.bfloat16).requires_grad_(True)
        f32 = lambda t: t.to(device).requires_grad_(True)
        self.D = D
        self.p = dict(embed=mk(D, dim, std=dim ** -0.5), norm=torch.ones(D, dtype=torch.bfloat16, device=device, requires_grad=True),
                      w_in=mk(2 * D, D, std=D ** -0.5), conv=mk(D, TAPS, std=TAPS ** -0.5), conv_bias=mk(D, std=0.1),
                      w_mix=mk(RANK + 2 * STATES, D, std=D ** -0.5), w_dt=mk(D, RANK, std=RANK ** -0.5),
                      w_out=mk(D, D, std=D ** -0.5), head=mk(classes, D, std=0.1 * D ** -0.5),
                      log_a=f32(torch.arange(1, STATES + 1).float().log().repeat(D, 1)), d=f32(torch.ones(D)),
                      dt_bias=f32(torch.log(torch.expm1(torch.exp(torch.rand(D, generator=g) * 4.6) * 1e-3))))

    def parameters(self):
        return list(self.p.values())

    def start(self, E, R, device="cuda"):
        """The memory before the first step: (inputs of the convolution, states of the scan)."""
        return (torch.zeros(E, R, TAPS - 1, self.D, dtype=torch.bfloat16, device=device),
                torch.zeros(E, R, self.D, STATES, device=device))

    def _run(self, obs, conv, scan):
        p = self.p
        e = obs.to(torch.bfloat16) @ p["embed"].T
        x, z = (ops.block_norm(e, p["norm"]) @ p["w_in"].T).split(self.D, -1)
        x = conv(x, p["conv"], p["conv_bias"])
        dt, b, c = (x @ p["w_mix"].T).split((RANK, STATES, STATES), -1)
        y = scan(x, dt @ p["w_dt"].T, -torch.exp(p["log_a"]), b, c, dict(d=p["d"], z=z, dt_bias=p["dt_bias"]))
        return ((e + y @ p["w_out"].T) @ p["head"].T).float()

    def rollout(self, obs, reset, memory):
        """obs [E, R, T, dim], reset [E, 1, T]: (logits [E, R, T, classes], the memory after the last step)."""
        after = []

        def conv(x, w, bias):
            y, s = ops.causal_conv(x, w, bias, state=memory[0], reset=reset)
            after.append(s)
            return y

        def scan(x, dt, a, b, c, more):
            y, s = ops.selective_scan(x, dt, a, b, c, state=memory[1], reset=reset, **more)
            after.append(s)
            return y

        return self._run(obs, conv, scan), after

    @torch.no_grad()
    def step(self, obs, reset, memory):
        """One control step: obs [E, R, dim], reset [E, 1]; the memory is updated in place."""
        return self._run(obs, lambda x, w, bias: ops.causal_conv_step(x, w, memory[0], bias, reset=reset),
                         lambda x, dt, a, b, c, more: ops.selective_scan_step(x, dt, a, b, c, memory[1], reset=reset, **more))


def main(envs=64, robots=16, rollouts=4, length=16, lr=0.02, verbose=True):
    wl = presets.workload(1)
    cfg = wl.config(traffic=(), msg_sizes=(200.0, 1500.0, 8192.0))
    net = ib.NetModule("L2", envs, robots, "cuda", cfg, seed=wl.seed, isaac=ib.IsaacNetCfg(
        radio="engine", obs_features=("aoi", "sinr", "queue_len", "last_delivered", "delay_history")))
    motion = presets.Motion(1, envs, robots, seed=wl.seed)
    classes, g = 1 + len(cfg.msg_sizes), torch.Generator(device="cuda").manual_seed(1)
    student = MemoryPolicy(net.obs_dim, classes)
    teacher = torch.randn(classes, net.obs_dim, generator=g, device="cuda")
    memory, seen = student.start(envs, robots), torch.zeros(envs, robots, net.obs_dim, device="cuda")
    net.reset()
    pos, fresh, log = motion.current(), torch.ones(envs, dtype=torch.bool, device="cuda"), []
    for k in range(rollouts):
        before = [m.clone() for m in memory]
        obs, flags, top, index = [], [], [], []
        for _ in range(length):
            o = net.obs().clone()
            seen = torch.where(fresh[:, None, None], 0.0, 0.8 * seen) + o          # what the teacher knows of earlier steps
            t = torch.topk(seen @ teacher.T, TOP)
            logits = student.step(o, fresh[:, None], memory)
            eng = net.eng
            u = ops.uniforms(eng.s0, robots, eng.env_id, eng.episode, net.clock, stream=100)
            net.submit(None, ib.TrafficRequest(ops.sample_logits(logits, u)[0]))
            net.step(None, pos.cuda())
            pos = motion.advance()
            obs.append(o), flags.append(fresh), top.append(t.values), index.append(t.indices)
            fresh = torch.rand(envs, generator=g, device="cuda") < 0.05            # episodes that end here
            if bool(fresh.any()):
                net.reset(fresh.nonzero()[:, 0])
        # the buffers were filled step by step: [T, E, ...] as [E, ..., T, ...]
        obs, flags = torch.stack(obs).permute(1, 2, 0, 3), torch.stack(flags).t()[:, None]
        top, index = (torch.stack(q).permute(1, 2, 0, 3) for q in (top, index))
        logits, _ = student.rollout(obs, flags, before)
        loss = ops.distill_loss(logits, top, index, temperature=2.0).mean()
        for p, gr in zip(student.parameters(), torch.autograd.grad(loss, student.parameters())):
            with torch.no_grad():
                p -= lr * gr
        log.append(float(loss.detach()))
        if verbose:
            print(f"rollout {k:3d}  distillation loss {log[-1]:.4f}")
    return log


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("envs", 64), ("robots", 16), ("rollouts", 4), ("length", 16)):
        ap.add_argument("--" + name, type=int, default=value)
    main(**vars(ap.parse_args()))
