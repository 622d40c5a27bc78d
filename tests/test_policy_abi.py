"""The policy operators' C ABI without a GPU: structure layouts, the statuses of refused calls (returned before anything
touches a device), and the Python entry points' refusal of CPU tensors."""
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

STRUCTS = {"InbNormArgs": nat.InbNormArgs, "InbDropoutArgs": nat.InbDropoutArgs, "InbSampleArgs": nat.InbSampleArgs,
           "InbFfnArgs": nat.InbFfnArgs}


def test_policy_struct_layouts_match_the_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "isaac_net_b200.h"', "int main(void) {"]
    for cname, cls in STRUCTS.items():
        lines.append(f'  printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    consts = ("INB_BF16", "INB_F16", "INB_F32", "INB_MAX_NORM_D", "INB_MAX_SAMPLE_V", "INB_MAX_SAMPLE_N", "INB_MAX_FFN",
              "INB_FFN_ROWS", "INB_MAX_NORM_LD", "INB_ACT_SILU", "INB_ACT_GELU")
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
    want = (nat.BF16, nat.F16, nat.F32, nat.MAX_NORM_D, nat.MAX_SAMPLE_V, nat.MAX_SAMPLE_N, nat.MAX_FFN,
            nat.FFN_ROWS, nat.MAX_NORM_LD, nat.ACTS["silu"], nat.ACTS["gelu"])
    assert [int(got[k]) for k in consts] == list(want)


def _norm(**kw):
    return nat.InbNormArgs(**{**dict(dtype=nat.F32, D=8, N=4, ldx=8, x=256, w=256, n=256), **kw})


def test_refused_calls_return_their_status():
    L = nat.lib()
    r = ctypes.byref
    norm = [(dict(D=0), -2), (dict(D=8193), -2), (dict(dtype=3), -2), (dict(N=-1), -2), (dict(x=None), -3),
            (dict(n=None), -3), (dict(gate=256), -3), (dict(h=256, y=256, ldh=8, gate=256, gate_rows=3), -4),
            (dict(N=0), 0)]
    for kw, rc in norm:
        assert L.inb_block_norm_fwd(r(_norm(**kw)), None) == rc, kw
    assert L.inb_block_norm_fwd(None, None) == -1
    assert L.inb_block_norm_bwd(r(_norm()), None) == -3
    assert L.inb_block_norm_bwd(r(_norm(stats=256, gx=256, gw=256, work=256, work_elems=1)), None) == -5
    d = lambda **kw: nat.InbDropoutArgs(**{**dict(dtype=nat.F32, threshold=1, E=2, n=4, env_id=256, x=256, y=256), **kw})
    for kw, rc in [(dict(threshold=65537), -2), (dict(E=-1), -2), (dict(n=1 << 34), -2), (dict(x=None), -3),
                   (dict(env_id=None), -3), (dict(E=0), 0), (dict(n=0), 0), (dict(E=1 << 31), -2)]:
        assert L.inb_dropout(r(d(**kw)), None) == rc, kw
    s = lambda **kw: nat.InbSampleArgs(**{**dict(dtype=nat.F32, V=8, N=4, ld=8, logits=256, u=256, token=256, logp=256),
                                          **kw})
    for kw, rc in [(dict(V=0), -2), (dict(V=(1 << 22) + 1), -2), (dict(N=(1 << 27) + 1), -2), (dict(u=None), -3),
                   (dict(logp=None), -3), (dict(N=0), 0)]:
        assert L.inb_sample(r(s(**kw)), None) == rc, kw
    f = lambda **kw: nat.InbFfnArgs(**{**dict(dtype=nat.BF16, D=8, F=8, N=4, ldx=8, ldwg=8, ldwu=8, ldwd=8, ldh=8, x=256,
                                              wg=256, wu=256, wd=256, y=256, h=256), **kw})
    for kw, rc in [(dict(dtype=nat.F32), -2), (dict(act=2), -2), (dict(ldh=9), -2), (dict(ldh=0), -2), (dict(F=0), -2),
                   (dict(x=None), -3), (dict(h=264), -3), (dict(g=256), -3), (dict(N=40, ldx=9), -5), (dict(N=0), 0)]:
        assert L.inb_gated_ffn_fwd(r(f(**kw)), None) == rc, kw
    assert L.inb_gated_ffn_bwd(r(f()), None) == -3


def test_work_sizes():
    L = nat.lib()
    size = nat.i64()
    a = nat.InbFfnArgs(dtype=nat.BF16, D=9, F=8, N=40, ldx=9, ldwg=16, ldwu=9, ldwd=8, ldh=8, x=256, wg=256, wu=256, wd=258)
    assert L.inb_gated_ffn_work(ctypes.byref(a), 0, ctypes.byref(size)) == 0
    assert size.value == 1280 + 256 + 256             # x, wu (rows of 9) and wd (base off 16 bytes), each padded
    a.N = 4                                           # few rows: the weights are read as they are
    assert L.inb_gated_ffn_work(ctypes.byref(a), 0, ctypes.byref(size)) == 0 and size.value == 0
    assert L.inb_gated_ffn_work(ctypes.byref(a), 0, None) == -1


def test_cpu_tensors_are_refused():
    x, w = torch.ones(4, 8), torch.ones(8)
    env = torch.arange(4)
    for f in (lambda: ops.block_norm(x, w), lambda: ops.counter_dropout(x, 0.5, 1, env),
              lambda: ops.sample_logits(x, w[:4]),
              lambda: ops.gated_ffn(x.bfloat16(), *(torch.ones(s).bfloat16() for s in ((16, 8), (16, 8), (8, 16))))):
        with pytest.raises(eng_mod.B200Unsupported):
            f()
