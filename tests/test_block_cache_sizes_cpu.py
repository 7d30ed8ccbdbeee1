"""Sizes of a block-scaled cache are whole numbers."""

import numpy as np
import pytest

from synthefy_nori_b200 import ops
from synthefy_nori_b200.inference.memory_policy import MemoryPolicy, block_footprint_gb, estimate_cache_gb, int8_footprint_gb


@pytest.mark.parametrize("kw", [dict(capacity=100.5), dict(head_dim=16.5), dict(batch=1.5), dict(heads=2.0), dict(block=64.0)])
def test_fractions_are_refused(kw):
    args = dict(batch=2, heads=2, capacity=100, head_dim=16, block=64) | kw
    with pytest.raises((TypeError, ValueError)):
        ops.block_cache(**args, device="cpu")


def test_whole_numbers_of_numpy():
    c = ops.block_cache(*(np.int64(x) for x in (2, 3, 100, 20)), device="cpu")
    assert c.k.shape == (2, 3, 128, 24) and c.head_dim == 20 and type(c.head_dim) is int


@pytest.mark.parametrize("dtype", ["bf16", "int8", "block_int8", "block_fp8"])
def test_shards_of_several_gpus_hold_int8(dtype):
    """The sharded rung has one form, int8 with a scale for each vector: it is sized and named as that."""
    table = dict(n_context_rows=100_000, n_groups=21, nlayers=26, embed_dim=448, head_dim=56, device_total_gb=20.0,
                 host_total_gb=0.0)
    got = MemoryPolicy(cache_dtype=dtype).resolve(**table, n_gpus=8)
    assert got.rung == "context_sharded_int8" and got.placement() == ("int8", "resident", None)
    assert got.resident_gb == pytest.approx(int8_footprint_gb(got.est_cache_gb, head_dim=56) / 8)
    # a budget that block scales would meet (1 + 4 / 3584) and a scale for each vector (1 + 4 / 56) does not
    tight = MemoryPolicy(cache_dtype=dtype, gpu_budget_absolute_gb=got.est_cache_gb / 16 * 1.03)
    assert tight.resolve(**table, n_gpus=8).rung == "subsample"


@pytest.mark.parametrize("rows", [1, 5, 127, 128, 129, 1000, 100_003])
@pytest.mark.parametrize("d", [16, 44, 56])
def test_the_policy_knows_the_capacity(rows, d):
    """What a context of any number of rows takes is what its buffers take: 128 rows at a time."""
    H, layers, tokens = 2, 3, 5
    cache = ops.block_cache(tokens, H, rows, d, device="meta")
    bf16 = estimate_cache_gb(n_context_rows=rows, n_groups=tokens, nlayers=layers, embed_dim=H * d)
    size = layers * cache.nbytes() / 2 ** 30
    assert block_footprint_gb(bf16, head_dim=d, n_context_rows=rows) == pytest.approx(size)
    table = dict(n_context_rows=rows, n_groups=tokens, nlayers=layers, embed_dim=H * d, head_dim=d, device_total_gb=100.0,
                 host_total_gb=0.0)
    for share, rung in ((1.001, "resident_int8"), (0.999, "subsample")):
        pol = MemoryPolicy(cache_dtype="block_int8", gpu_budget_absolute_gb=size * share).resolve(**table)
        assert pol.rung == rung
        if rung == "resident_int8":
            assert pol.resident_gb == pytest.approx(size)
        else:  # whole capacities that fit, one at least
            kept = rows - pol.dropped_context_rows
            assert kept == max(1, -(-rows // 128) * 128 - 128)
