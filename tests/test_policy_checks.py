"""Argument checks of the policy operators that need no GPU."""
import ctypes
import importlib

import pytest
import torch

nat = importlib.import_module("isaac-net_b200._native")
ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")


class On(torch.Tensor):
    """A tensor that says which device it is on and gives no address: what a check lets pass ends in a RuntimeError."""
    device = property(lambda self: self.where)
    is_cuda = property(lambda self: self.where.type == "cuda")

    def data_ptr(self):
        raise RuntimeError("went on to the launch")


def ids(where="cuda:0", shape=(4,), dtype=torch.int64):
    t = torch.zeros(shape, dtype=dtype).as_subclass(On)
    t.where = torch.device(where)
    return t


def test_uniforms_refuses_what_counter_dropout_refuses():
    env = ids()
    for kind, args, kw in [
            (ValueError, (1, 8, env, ids("cuda:1")), {}), (ValueError, (1, 8, env, None, ids("cuda:1")), {}),
            (eng_mod.B200Unsupported, (1, 8, env, ids("cpu")), {}), (eng_mod.B200Unsupported, (1, 8, ids("cpu")), {}),
            (TypeError, (1, 8, env, ids(dtype=torch.int32)), {}), (TypeError, (1, 8, ids(dtype=torch.float32)), {}),
            (TypeError, (1, 8, None), {}), (TypeError, (1, 8, env, 3), {}),
            (ValueError, (1, 8, env, ids(shape=(5,))), {}), (ValueError, (1, 8, ids(shape=(4, 2))), {}),
            (ValueError, (-1, 8, env), {}), (ValueError, (1 << 32, 8, env), {}), (ValueError, (1, 8, env), dict(stream=-1)),
            (eng_mod.B200Unsupported, (1, -1, env), {}), (eng_mod.B200Unsupported, (1, 1 << 30, env), {})]:
        with pytest.raises(kind, match="env_id|episode|ctr|32-bit|draws"):
            ops.uniforms(*args, **kw)
            pytest.fail(f"{args}, {kw} was not refused")


def test_block_norm_entries_refuse_strides_that_32_bits_cannot_hold():
    """At the C entry points, which callers of other languages reach without the Python layer's checks; what a check lets
    pass ends at a NULL output (-3) or at the scratch that is too small (-5), not in a launch."""
    L, most = nat.lib(), nat.MAX_NORM_LD
    good = dict(dtype=nat.F32, D=8, N=4, ldx=8, x=256, w=256)
    back = dict(good, h=256, ldh=8, gy=256, ldgy=8, gn=256, ldgn=8, stats=256, gx=256, gw=256, gh=256, work=256)
    for base, call, passed in ((good, L.inb_block_norm_fwd, -3), (back, L.inb_block_norm_bwd, -5)):
        for name in [k for k in base if k.startswith("ld")]:
            for ld, rc in ((0, passed), (8, passed), (most, passed), (most + 1, -2), (1 << 32, -2), ((1 << 32) + 8, -2), (-8, -2)):
                assert call(ctypes.byref(nat.InbNormArgs(**dict(base, **{name: ld}))), None) == rc, (name, ld)
    absent = nat.InbNormArgs(**dict(good, ldh=1 << 40, ldgy=-1))          # strides of tensors that are not given
    assert L.inb_block_norm_fwd(ctypes.byref(absent), None) == -3
