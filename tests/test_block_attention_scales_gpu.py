"""Attention over a block-scaled cache whose values differ by more than fp32's exponents from block to block: the sum
of the weights and the log-sum-exp do not depend on V."""

import pytest
import torch

from test_block_attention_gpu import check

pytestmark = pytest.mark.gpu

SIZES = [(1e30, 0.0), (0.0, 1e30), (1e30, 1.0, 0.0), (1e18, 0.0, 1e-12, 1e3), (1e25, 1e-10), (0.0, 1e-12, 1e33)]


@pytest.mark.parametrize("n,rows", [(1, 512), (1, 20000), (1, 70001), (12, 3000), (200, 512), (300, 5000)])
@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_sums_reach_past_the_scales(n, rows, sizes, dtype):
    """Blocks of 64 rows in turn (runs of 1024 rows in longer contexts, so that warps, clusters and parts that are
    joined each hold one size); keys of all sizes have scores alike."""
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(n + rows)
    run = 64 if rows < 1000 else 1024
    which = torch.arange(rows, device="cuda") // run % len(sizes)
    size = torch.tensor(sizes, device="cuda")[which].view(1, -1, 1, 1)
    k, v = (torch.randn(1, rows, 2, 56, device="cuda", generator=g) for _ in "kv")
    cache = ops.block_cache(1, 2, rows, 56, dtype=dtype, block=64)
    ops.block_cache_write(cache, k, v * size)
    q = (2 * torch.randn(1, n, 2, 56, device="cuda", generator=g)).to(torch.bfloat16)
    o, lse = ops.block_cache_attention(q, cache, rows, return_lse=True)
    check(q, cache, [rows], o, lse)
