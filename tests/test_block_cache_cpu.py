"""Block-scaled context cache without a GPU: refusals, sizes, and the settings that choose it."""

import pytest
import torch

from synthefy_nori_b200 import ops
from synthefy_nori_b200.inference.memory_policy import MemoryPolicy, block_footprint_gb, int8_footprint_gb

needs_lib = pytest.mark.skipif(not ops.native_available(), reason="the extension is not built")


@pytest.mark.parametrize("kw", [dict(dtype=torch.uint8), dict(dtype=torch.float8_e5m2), dict(block=16), dict(block=48),
                                dict(head_dim=0), dict(head_dim=65), dict(batch=-1), dict(capacity=-1)])
def test_sizes_that_are_no_cache(kw):
    args = dict(batch=2, heads=2, capacity=100, head_dim=16) | kw
    with pytest.raises(ValueError):
        ops.block_cache(**args, device="cpu")


@pytest.mark.parametrize("capacity,rows", [(0, 128), (1, 128), (128, 128), (129, 256), (1000, 1024)])
@pytest.mark.parametrize("d,width", [(1, 8), (8, 8), (44, 48), (56, 56), (64, 64)])
def test_cache_sizes(capacity, rows, d, width):
    for dtype in ops.BLOCK_CACHE_TYPES:
        for block in (32, 64, 128):
            c = ops.block_cache(3, 2, capacity, d, dtype=dtype, block=block, device="cpu")
            assert c.k.shape == c.v.shape == (3, 2, rows, width) and c.k.dtype == c.v.dtype == dtype
            assert c.k_scale.shape == c.v_scale.shape == (3, 2, rows // block) and c.k_scale.dtype == torch.float32
            assert (c.block, c.capacity, c.head_dim) == (block, rows, d)
            assert c.nbytes() == 2 * 3 * 2 * (rows * width + 4 * rows // block)


def test_cpu_tensors_are_refused():
    c = ops.block_cache(1, 2, 128, 16, device="cpu")
    x = torch.zeros(1, 4, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.block_cache_write(c, x, x)
    with pytest.raises(ValueError):
        ops.block_cache_read(c)
    with pytest.raises(ValueError):
        ops.block_cache_attention(x, c, 4)


def _parts(**kw):
    c = ops.block_cache(1, 2, 256, 16, block=64, device="cpu")
    return (dict(k=c.k, v=c.v, ks=c.k_scale, vs=c.v_scale, d=16) | kw).values()


@needs_lib
@pytest.mark.parametrize("change", [
    lambda c: dict(k=c.k.view(torch.uint8)),  # another type
    lambda c: dict(v=c.v.view(torch.float8_e4m3fn)),  # two types
    lambda c: dict(v=c.v[:, :1].contiguous()),
    lambda c: dict(k=c.k[:, :, :200].contiguous(), v=c.v[:, :, :200].contiguous()),  # no multiple of 128 rows
    lambda c: dict(k=c.k[0], v=c.v[0]),
    lambda c: dict(k=c.k.transpose(1, 2)),
    lambda c: dict(ks=c.k_scale.double()),
    lambda c: dict(ks=c.k_scale[:, :, :3].contiguous(), vs=c.v_scale[:, :, :3].contiguous()),  # no block of 32, 64, 128
    lambda c: dict(ks=torch.zeros(1, 2, 1), vs=torch.zeros(1, 2, 1)),  # 256 rows a block
    lambda c: dict(ks=torch.zeros(1, 2, 16), vs=torch.zeros(1, 2, 16)),  # 16
    lambda c: dict(ks=torch.zeros(2, 2, 4), vs=torch.zeros(2, 2, 4)),
    lambda c: dict(d=0), lambda c: dict(d=17), lambda c: dict(d=8), lambda c: dict(d=65),
    lambda c: {},  # not on a GPU
])
def test_cache_tensors_that_do_not_fit_are_refused(change):
    c = ops.block_cache(1, 2, 256, 16, block=64, device="cpu")
    with pytest.raises(RuntimeError, match="block_cache_read"):
        ops.lib().block_cache_read(*_parts(**change(c)), 0, 4, torch.bfloat16)


def test_memory_policy_of_block_caches():
    """The block-scaled types take the place of int8 on every rung, and their size decides it."""
    table = dict(n_context_rows=100_000, n_groups=21, nlayers=26, embed_dim=448, head_dim=56)
    for dtype in ("block_int8", "block_fp8"):
        pol = MemoryPolicy(cache_dtype=dtype)
        got = pol.resolve(**table, device_total_gb=178.0)
        assert got.rung == "resident_int8" and got.placement() == (dtype, "resident", None)
        small = pol.resolve(**table, device_total_gb=40.0, host_total_gb=500.0)
        assert small.rung == "offload_int8" and small.placement() == (dtype, "offload", None)
        stream = MemoryPolicy(cache_dtype=dtype, stream_context=True).resolve(**table, device_total_gb=40.0, host_total_gb=500.0)
        assert stream.rung == "stream_int8" and stream.placement()[0] == dtype and stream.placement()[1] == "stream"
    assert MemoryPolicy().resolve(**table, device_total_gb=178.0).placement()[0] in ("bf16", "int8")
    # 1 + 1 / 896 of half the bf16 cache at width 56, where a scale for each vector takes 1 + 4 / 56
    assert block_footprint_gb(2.0, head_dim=56) == pytest.approx(1.0 + 4 / (64 * 56))
    assert block_footprint_gb(2.0, head_dim=44) == pytest.approx(48 / 44 + 4 / (64 * 44))
    assert block_footprint_gb(2.0, head_dim=56) < int8_footprint_gb(2.0, head_dim=56)
    with pytest.raises(ValueError):
        MemoryPolicy(cache_dtype="block_int4")


@pytest.mark.parametrize("dtype", ["block_int8", "block_fp8"])
def test_block_caches_need_the_native_path(dtype):
    from synthefy_nori_b200.inference.predictor import NoriPredictor
    from synthefy_nori_b200.models.config import preset_config
    from synthefy_nori_b200.utils.loading import build_model

    model = build_model(preset_config("nori-tiny")).eval()
    x, y = torch.randn(1, 20, 4), torch.randn(1, 20)
    with pytest.raises(NotImplementedError, match="CUDA"):
        model.build_context_cache(x, y, cache_dtype=dtype)
    with pytest.raises(ValueError, match="cache_dtype"):
        model.build_context_cache(x, y, cache_dtype="block_int4")
    assert NoriPredictor(model, "cpu", cache_dtype=dtype).cache_dtype == dtype
    with pytest.raises(ValueError, match="cache_dtype"):
        NoriPredictor(model, "cpu", cache_dtype="fp8")
