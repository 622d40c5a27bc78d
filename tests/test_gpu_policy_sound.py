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


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("v", [385, 511, 1001, 1002, 1003, 1535, 4095])
def test_sample_logits_rows_that_end_inside_an_access(v, dtype):
    """Rows that a block keeps in shared memory, at every remainder of a 16-byte access: masked up to the last element, and
    with the last element alone."""
    from test_gpu_policy_ops import check_sample
    g = gen(v)
    logits, u = (rn(g, 5, v) * 2).to(dtype), torch.rand(5, generator=g, device="cuda")
    ends = torch.rand(5, v, generator=g, device="cuda") < 0.5
    ends[:, -1] = True
    last = torch.zeros(5, v, dtype=torch.bool, device="cuda")
    last[:, -1] = True
    for mask in (None, ends, last):
        for k, p in ((0, 0.9), (200, 0.8), (v - 1, 1.0)):
            check_sample(logits, u, 1.0, k, p, 0.0, mask=mask)
