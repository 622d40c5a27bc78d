"""The policy operators where a fault of one tile, row or call could reach another.  Tolerances as in the operators' own
test files."""
import importlib

import pytest
import torch

ops = importlib.import_module("isaac-net_b200.policy_ops")
eng_mod = importlib.import_module("isaac-net_b200.engine")

pytestmark = pytest.mark.gpu
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
