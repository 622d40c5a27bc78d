"""Argument checks of the policy operators that need no GPU."""
import importlib

import pytest
import torch
from torch._subclasses import FakeTensorMode

ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")


def test_uniforms_refuses_what_counter_dropout_refuses():
    """On tensors without storage, so a call that went on would end in an error of another kind, not in a launch."""
    with FakeTensorMode():
        ids = lambda device="cuda:0", shape=(4,), dtype=torch.int64: torch.zeros(shape, dtype=dtype, device=device)
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
