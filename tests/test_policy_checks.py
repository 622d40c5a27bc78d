"""Argument checks of the policy operators that need no GPU."""
import importlib

import pytest
import torch

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
