"""Context cache in 8 bits with block scales: rows written and read back, against the same formulas in
64 bits (scales and roundings in 32, as they are defined)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def _f32(x):
    return torch.tensor(x, dtype=torch.float32)


def _code(y, dtype):
    """fp32 values to codes, ties to even."""
    top = TOP[dtype]
    y = y.clamp(-top, top)
    return (y.round() if dtype == torch.int8 else y).to(dtype)


def written(codes, scales, x, start, count, block, dtype):
    """The definition, on the CPU: ``codes`` [cap, W], ``scales`` [blocks] and new rows ``x`` [n, D] of one
    sequence and head, updated in place."""
    cap, d = codes.shape[0], x.shape[1]
    lo, hi = max(start, 0), min(start + max(min(count, x.shape[0]), 0), cap)
    for blk in range(lo // block, -(-hi // block) if hi > lo else 0):
        r0, r1 = max(blk * block, lo), min((blk + 1) * block, hi)
        rows = x[r0 - start : r1 - start].float()
        s = torch.maximum(rows.abs().max(), _f32(1e-12)) / _f32(TOP[dtype])
        old = scales[blk].clone() if r0 > blk * block else _f32(0.0)
        s = torch.maximum(s, old)  # a NaN stays
        inv = _f32(1.0) / s
        if r0 > blk * block and not torch.equal(s, old):
            kept = codes[blk * block : r0]
            kept.copy_(_code(kept.float() * (old * inv), dtype))
        codes[r0:r1, :d] = _code(rows * inv, dtype)
        codes[r0:r1, d:] = _code(torch.zeros(r1 - r0, codes.shape[1] - d), dtype)
        scales[blk] = s


def _check(cache, ref, rows=None):
    for got, want, gs, ws in ((cache.k, ref[0], cache.k_scale, ref[2]), (cache.v, ref[1], cache.v_scale, ref[3])):
        assert torch.equal(gs.cpu().nan_to_num(nan=-1.0), ws.nan_to_num(nan=-1.0))
        assert torch.equal(got.cpu().view(torch.int8), want.view(torch.int8))


def _reference(cache):
    return [t.cpu().clone() for t in cache[:4]]


def _write_reference(ref, cache, k, v, starts, counts):
    k, v = k.cpu(), v.cpu()
    if k.dim() == 5:
        k, v = k.flatten(0, 1), v.flatten(0, 1)
    for b in range(k.shape[0]):
        for h in range(k.shape[2]):
            for codes, scales, x in ((ref[0], ref[2], k), (ref[1], ref[3], v)):
                written(codes[b, h], scales[b, h], x[b, :, h], starts[b], counts[b], cache.block, cache.k.dtype)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("block,d,n,start", [(32, 8, 1, 0), (32, 44, 97, 0), (64, 56, 130, 0), (64, 56, 3, 61),
                                             (64, 64, 200, 63), (128, 33, 300, 100), (128, 1, 129, 127), (32, 20, 384, 0)])
def test_write_matches_definition(dtype, src, block, d, n, start):
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(7 * d + n)
    cache = ops.block_cache(2, 3, 500, d, dtype=dtype, block=block)
    ref = _reference(cache)
    # what is there before: smaller rows, so that blocks which stay have to be quantised again
    if start:
        old = 0.3 * torch.randn(2, start, 3, d, device="cuda", generator=g)
        ops.block_cache_write(cache, old, -old)
        _write_reference(ref, cache, old, -old, [0, 0], [start, start])
    k, v = (torch.randn(2, n, 3, d, device="cuda", generator=g).to(src) for _ in "kv")
    ops.block_cache_write(cache, k, v, start=start)
    _write_reference(ref, cache, k, v, [start] * 2, [n] * 2)
    _check(cache, ref)


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_write_row_by_row(dtype):
    """Single rows appended: scales grow, earlier rows are quantised again, smaller rows change nothing."""
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(1, 2, 128, 24, dtype=dtype, block=32)
    ref = _reference(cache)
    g = torch.Generator(device="cuda").manual_seed(3)
    for i in range(40):
        k = torch.randn(1, 1, 2, 24, device="cuda", generator=g).to(torch.bfloat16) * (1 + i % 7)
        v = torch.randn(1, 1, 2, 24, device="cuda", generator=g).to(torch.bfloat16)
        ops.block_cache_write(cache, k, v, start=i)
        _write_reference(ref, cache, k, v, [i], [1])
    _check(cache, ref)


def test_write_ragged_on_the_device():
    """Each sequence at its own place; rows outside the capacity and behind a count are not written."""
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(6, 2, 256, 40, block=64)
    g = torch.Generator(device="cuda").manual_seed(5)
    base = torch.randn(6, 256, 2, 40, device="cuda", generator=g)
    ops.block_cache_write(cache, base, base)
    ref = _reference(cache)
    k, v = (3 * torch.randn(6, 100, 2, 40, device="cuda", generator=g) for _ in "kv")
    starts, counts = [0, 10, 200, 255, -20, 300], [0, 100, 100, 5, 60, 100]
    ops.block_cache_write(cache, k, v, start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                          counts=torch.tensor(counts, dtype=torch.int32, device="cuda"))
    _write_reference(ref, cache, k, v, starts, counts)
    _check(cache, ref)


@pytest.mark.parametrize("shift", [0, 1, 4])
def test_write_strided_rows(shift):
    """K and V as columns of one projection, two batch dimensions, any alignment."""
    from synthefy_nori_b200 import ops

    B, N, T, H, D = 2, 70, 3, 2, 24
    y = torch.randn(B * N * T * 5 * H * D + 8, device="cuda").to(torch.bfloat16)[shift:][: B * N * T * 5 * H * D]
    y = y.view(B, N, T, 5, H, D)
    k, v = (y[:, :, :, i].permute(0, 2, 1, 3, 4) for i in (3, 4))
    cache = ops.block_cache(B * T, H, N, D, block=32)
    ref = _reference(cache)
    ops.block_cache_write(cache, k, v)
    _write_reference(ref, cache, k, v, [0] * 6, [N] * 6)
    _check(cache, ref)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
def test_non_finite_values_make_their_block_nan(bad, dtype, src):
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(1, 2, 128, 16, dtype=dtype, block=32)
    k = torch.randn(1, 128, 2, 16, device="cuda").to(src)
    v = k.clone()
    k[0, 40, 1, 3] = bad
    ops.block_cache_write(cache, k, v)
    ko, vo = ops.block_cache_read(cache)
    nan = torch.zeros(1, 128, 2, 16, dtype=torch.bool, device="cuda")
    nan[0, 32:64, 1] = True
    assert torch.equal(ko.isnan(), nan) and not vo.isnan().any()
    # a later row in the block does not hide it
    ops.block_cache_write(cache, torch.ones(1, 1, 2, 16, device="cuda"), torch.ones(1, 1, 2, 16, device="cuda"), start=50)
    assert ops.block_cache_read(cache)[0][0, 32:64, 1].isnan().all()


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d,start,end", [(8, 0, 256), (44, 17, 101), (33, 5, 6), (56, 0, 0), (64, 100, 256), (1, 3, 200)])
def test_read_is_code_times_scale(dtype, out, d, start, end):
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(3, 2, 256, d, dtype=dtype, block=64)
    k, v = (torch.randn(3, 256, 2, d, device="cuda") for _ in "kv")
    ops.block_cache_write(cache, k, v)
    for got, code, scale in zip(ops.block_cache_read(cache, start, end, dtype=out), cache[:2], cache[2:4]):
        want = code.float() * scale.repeat_interleave(64, 2)[..., None]
        want = want[:, :, start:end, :d].transpose(1, 2).to(out)
        assert got.shape == want.shape and torch.equal(got, want)


def test_round_trip_error():
    """Half a step of the block's scale (int8), half a step of the value (e4m3: 2^-4, or 2^-10 of a scale's step
    for the smallest)."""
    from synthefy_nori_b200 import ops

    x = torch.randn(2, 1000, 2, 56, device="cuda")
    for dtype in ops.BLOCK_CACHE_TYPES:
        cache = ops.block_cache(2, 2, 1000, 56, dtype=dtype)
        ops.block_cache_write(cache, x, x)
        k, _ = ops.block_cache_read(cache, 0, 1000, dtype=torch.float32)
        step = cache.k_scale.repeat_interleave(64, 2)[:, :, :1000, None].transpose(1, 2)
        bound = 0.5 * step if dtype == torch.int8 else torch.maximum(x.abs() * 2.0 ** -4, step * 2.0 ** -10)
        # plus the fp32 roundings of x / s and code * s
        assert ((k - x).abs() <= bound + x.abs() * 2.0 ** -22).all()


def test_zero_rows_and_empty_sizes():
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(2, 2, 128, 16)
    z = torch.zeros(2, 100, 2, 16, device="cuda")
    ops.block_cache_write(cache, z, z)
    assert not ops.block_cache_read(cache, 0, 100)[0].any()
    ops.block_cache_write(cache, z[:, :0], z[:, :0], start=100)  # no rows: nothing happens
    empty = ops.block_cache(0, 2, 128, 16)
    ops.block_cache_write(empty, z[:0], z[:0])
    assert ops.block_cache_read(empty, 0, 5)[0].shape == (0, 5, 2, 16)


def test_write_captured_and_replayed():
    """A captured append at a device position: replays follow the position tensor."""
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(3, 2, 128, 32, block=32)
    ref = _reference(cache)
    k, v = (torch.zeros(3, 1, 2, 32, device="cuda") for _ in "kv")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    ops.block_cache_write(cache, k, v, start=pos)
    _write_reference(ref, cache, k, v, [0] * 3, [1] * 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.block_cache_write(cache, k, v, start=pos)
    for i in range(1, 50):
        x = torch.randn(2, 3, 1, 2, 32, device="cuda") * i
        k.copy_(x[0])
        v.copy_(x[1])
        pos.fill_(i)
        graph.replay()
        _write_reference(ref, cache, x[0], x[1], [i] * 3, [1] * 3)
    _check(cache, ref)


def test_versions_follow_writes():
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(1, 1, 128, 8)
    before = [t._version for t in cache[:4]]
    ops.block_cache_write(cache, torch.ones(1, 4, 1, 8, device="cuda"), torch.ones(1, 4, 1, 8, device="cuda"))
    assert all(t._version > b for t, b in zip(cache[:4], before))
