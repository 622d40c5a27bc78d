"""The C ABI of the policy's memory and of distill_loss without a GPU: structure layouts, the statuses of refused calls
(returned before anything touches a device), sizes of scratch, and the Python entry points' refusal of CPU tensors."""
import ctypes
import importlib
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
nat = importlib.import_module("isaac-net_b200._native")
ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

STRUCTS = {"InbSeq": nat.InbSeq, "InbReset": nat.InbReset, "InbConvArgs": nat.InbConvArgs, "InbScanArgs": nat.InbScanArgs,
           "InbDistillArgs": nat.InbDistillArgs}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "isaac_net_b200.h"', "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    consts = ("INB_MAX_MEMORY_C", "INB_MAX_MEMORY_S", "INB_MAX_SCAN_N", "INB_MAX_DISTILL_K")
    lines += [f'  printf("{c} %d\\n", (int){c});' for c in consts] + ["  return 0;", "}"]
    c, exe = tmp_path / "layout.c", tmp_path / "layout"
    c.write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(exe)], check=True, capture_output=True, text=True)
               .stdout.strip().splitlines())
    for cname, cls in STRUCTS.items():
        assert int(got[cname]) == ctypes.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"
    assert [int(got[k]) for k in consts] == [nat.MAX_MEMORY_C, nat.MAX_MEMORY_S, nat.MAX_SCAN_N, nat.MAX_DISTILL_K]


def seq(p=256, s=64, t=8):
    return nat.InbSeq(p, s, t)


def conv(**kw):
    return nat.InbConvArgs(**{**dict(dtype=nat.F32, act=0, C=8, K=4, S=3, T=5, x=seq(), y=seq(), w=256), **kw})


def scan(**kw):
    d = dict(dtype=nat.F32, C=8, N=4, S=3, T=5, a=256)
    d.update({k: seq() for k in ("x", "dt", "b", "c", "y")})
    return nat.InbScanArgs(**{**d, **kw})


def distill(**kw):
    return nat.InbDistillArgs(**{**dict(dtype=nat.F32, teacher_dtype=nat.F32, V=8, K=2, N=4, ld=8, logits=256, teacher=256, index=256,
                                        tau=1.0, loss=256), **kw})


def test_refused_calls_return_their_status():
    L, r = nat.lib(), ctypes.byref
    none = seq(None)
    for kw, rc in [(dict(dtype=3), -2), (dict(dtype=-1), -2), (dict(act=1), -2), (dict(act=-2), -2), (dict(C=0), -2),
                   (dict(C=nat.MAX_MEMORY_C + 1), -2), (dict(K=1), -2), (dict(K=5), -2), (dict(S=-1), -2), (dict(T=-1), -2),
                   (dict(S=nat.MAX_MEMORY_S + 1), -2), (dict(T=nat.MAX_MEMORY_S + 1), -2),
                   (dict(reset=nat.InbReset(256, 0, 1, 1)), -2), (dict(reset=nat.InbReset(256, 1 << 31, 1, 1)), -2),
                   (dict(x=none), -3), (dict(y=none), -3), (dict(w=None), -3), (dict(S=0), 0), (dict(T=0), 0)]:
        assert L.inb_causal_conv_fwd(r(conv(**kw)), None) == rc, kw
    assert L.inb_causal_conv_fwd(None, None) == -1 and L.inb_causal_conv_bwd(None, None) == -1
    back = dict(gy=seq(), gx=seq(), gw=256)
    for kw, rc in [(dict(gy=none), -3), (dict(gx=none), -3), (dict(gw=None), -3), ({}, -5), (dict(work=256, work_elems=1), -5),
                   (dict(S=0), 0)]:
        assert L.inb_causal_conv_bwd(r(conv(**{**back, **kw})), None) == rc, kw
    for kw, rc in [(dict(dtype=3), -2), (dict(C=0), -2), (dict(N=0), -2), (dict(N=65), -2), (dict(S=-1), -2), (dict(T=-1), -2),
                   (dict(S=1 << 25, C=1 << 10), -2), (dict(reset=nat.InbReset(256, 0, 1, 1)), -2), (dict(x=none), -3),
                   (dict(dt=none), -3), (dict(b=none), -3), (dict(c=none), -3), (dict(y=none), -3), (dict(a=None), -3),
                   (dict(T=0), 0), (dict(T=4000), -5), (dict(kept=264), -3), (dict(work=260), -3)]:
        assert L.inb_selective_scan_fwd(r(scan(**kw)), None) == rc, kw
    back = {k: seq() for k in ("gy", "gx", "gdt", "gb", "gc")}
    for kw, rc in [(dict(gy=none), -3), (dict(gx=none), -3), (dict(gdt=none), -3), (dict(gb=none), -3), (dict(gc=none), -3), ({}, -3),
                   (dict(ga=256, z=seq()), -3), (dict(ga=256, T=9), -3), (dict(ga=256), -5), (dict(ga=256, T=9, kept=256), -5), (dict(ga=256, T=9, kept=264), -3),
                   (dict(S=0), 0)]:
        assert L.inb_selective_scan_bwd(r(scan(**{**back, **kw})), None) == rc, kw
    for kw, rc in [(dict(dtype=3), -2), (dict(teacher_dtype=-1), -2), (dict(V=0), -2), (dict(V=(1 << 22) + 1), -2), (dict(K=0), -2),
                   (dict(K=1025), -2), (dict(N=-1), -2), (dict(tau=0.0), -2), (dict(tau=-1.0), -2), (dict(tau=float("nan")), -2),
                   (dict(tau=float("inf")), -2), (dict(logits=None), -3), (dict(teacher=None), -3), (dict(index=None), -3),
                   (dict(loss=None), -3), (dict(stats=264), -3), (dict(N=0), 0)]:
        assert L.inb_distill_fwd(r(distill(**kw)), None) == rc, kw
    for kw, rc in [(dict(), -3), (dict(stats=256), -3), (dict(stats=256, gloss=256), -3), (dict(N=0), 0)]:
        assert L.inb_distill_bwd(r(distill(**kw)), None) == rc, kw


def test_sizes_of_scratch():
    L, r, n = nat.lib(), ctypes.byref, nat.i64()
    assert L.inb_selective_scan_kept(r(scan(T=8)), r(n)) == 0 and n.value == 0
    assert L.inb_selective_scan_kept(r(scan(T=17, N=5)), r(n)) == 0 and n.value == 3 * 2 * 8 * 8       # S, steps 8 and 16, C, N up to 8
    assert L.inb_selective_scan_work(r(scan(T=1)), 0, r(n)) == 0 and n.value == 0
    assert L.inb_selective_scan_work(r(scan(T=4000)), 0, r(n)) == 0 and n.value > 0
    assert L.inb_selective_scan_work(r(scan(S=1 << 20, T=4000)), 0, r(n)) == 0 and n.value == 0         # sequences enough
    assert L.inb_selective_scan_work(r(scan()), 1, r(n)) == 0 and n.value >= 3 * 8 * (4 + 2)
    assert L.inb_causal_conv_work(r(conv()), r(n)) == 0 and n.value >= 8 * 5
    assert L.inb_causal_conv_work(r(conv()), None) == -1


def test_cpu_tensors_are_refused():
    x, w, s = torch.ones(2, 5, 8), torch.ones(8, 4), torch.zeros(2, 3, 8)
    b, a, h = torch.ones(2, 5, 4), torch.ones(8, 4), torch.zeros(2, 8, 4)
    for f in (lambda: ops.causal_conv(x, w), lambda: ops.causal_conv_step(x[:, 0], w, s), lambda: ops.selective_scan(x, x, a, b, b),
              lambda: ops.selective_scan_step(x[:, 0], x[:, 0], a, b[:, 0], b[:, 0], h),
              lambda: ops.distill_loss(x, x[..., :2], torch.zeros(2, 5, 2, dtype=torch.long))):
        with pytest.raises(eng_mod.B200Unsupported):
            f()
    with pytest.raises(ValueError):
        ops.causal_conv(x, w, act="relu")
