"""Block-scaled caches at the calls that are allowed and rarely made."""

import math
import random

import pytest
import torch

from test_block_attention_gpu import check, make, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(48))
def test_drawn_sizes(seed):
    """Sequences, heads, groups, rows, widths, blocks and lengths drawn together, the capacity far above the
    lengths in some (so that the keys are split further than they reach)."""
    from synthefy_nori_b200 import ops

    r = random.Random(seed)
    b, h, group = r.choice([1, 2, 5, 37]), r.choice([1, 2, 3, 8]), r.choice([1, 1, 2, 5])
    d, n = r.randint(1, 64), r.choice([1, 2, 7, 31, 33, 96, 128, 255, 256, 257, 290, 520])
    rows = r.choice([1, 5, 64, 127, 129, 300, 1100, 2600])
    if b * h * group * n * rows > 3e8:
        b = 1
    cache, g = make(b, h, rows, d, r.choice(ops.BLOCK_CACHE_TYPES), r.choice([32, 64, 128]), seed=seed)
    if r.random() < 0.3:  # room behind what is there
        big = ops.block_cache(b, h, rows + 20000, d, dtype=cache.k.dtype, block=cache.block)
        for dst, src in zip(big[:4], cache[:4]):
            dst[:, :, : src.shape[2]] = src
        cache = big
    q = (2 * torch.randn(b, n, h * group, d, device="cuda", generator=g)).to(r.choice([torch.bfloat16, torch.float16]))
    if r.random() < 0.3:  # head-major memory
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    lengths = [r.choice([0, 1, rows // 2, rows]) for _ in range(b)]
    where = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    scale = r.choice([None, 0.05, 1.0 / math.sqrt(d)])
    o, lse = ops.block_cache_attention(q, cache, where, scale=scale, return_lse=True)
    keep = max(rows, 1)
    # (the oracle reads what is there alone)
    part = type(cache)(*(t[:, :, : -(-keep // 128) * 128 // (1 if t.dim() == 4 else cache.block)].contiguous()
                         for t in cache[:4]), d)
    check(q, part, lengths, o, lse, scale)


@pytest.mark.parametrize("n", [1, 200])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_blocks_that_were_never_written(n, dtype):
    """They hold zeros: scores 0, values 0."""
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(2, 2, 640, 40, dtype=dtype, block=32)
    g = torch.Generator(device="cuda").manual_seed(n)
    k, v = (torch.randn(2, 70, 2, 40, device="cuda", generator=g) for _ in "kv")
    ops.block_cache_write(cache, k, v, start=200)
    q = torch.randn(2, n, 2, 40, device="cuda", generator=g).to(torch.bfloat16)
    o, lse = ops.block_cache_attention(q, cache, 600, return_lse=True)
    check(q, cache, [600, 600], o, lse)
    o, lse = ops.block_cache_attention(q, cache, 150, return_lse=True)  # none of them
    assert not o.any() and (lse - math.log(150)).abs().max() <= 2.0 ** -13


@pytest.mark.parametrize("n", [1, 200])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_blocks_of_very_different_sizes(n, dtype):
    """Values of 1e-12, 1 and 1e6 in neighbouring blocks."""
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(n)
    size = torch.tensor([1e-12, 1.0, 1e6, 1e-5], device="cuda").repeat_interleave(64).view(1, -1, 1, 1)
    k, v = (torch.randn(2, 256, 2, 56, device="cuda", generator=g) for _ in "kv")
    cache = ops.block_cache(2, 2, 256, 56, dtype=dtype, block=64)
    ops.block_cache_write(cache, k, v * size)
    q = torch.randn(2, n, 2, 56, device="cuda", generator=g).to(torch.bfloat16)
    for length in (64, 128, 256):
        o, lse = ops.block_cache_attention(q, cache, length, return_lse=True)
        check(q, cache, [length] * 2, o, lse)


def test_broadcast_inputs():
    """Keys that all heads share and a value row for all rows, as views without memory of their own."""
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(0)
    k = torch.randn(2, 100, 1, 24, device="cuda", generator=g).expand(-1, -1, 3, -1)
    v = torch.randn(2, 1, 3, 24, device="cuda", generator=g).expand(-1, 100, -1, -1)
    a, b = (ops.block_cache(2, 3, 100, 24) for _ in "ab")
    ops.block_cache_write(a, k, v)
    ops.block_cache_write(b, k.contiguous(), v.contiguous())
    assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4]))
    q = torch.randn(2, 1, 3, 24, device="cuda", generator=g).to(torch.bfloat16).expand(-1, 40, -1, -1)
    assert torch.equal(ops.block_cache_attention(q, a, 100), ops.block_cache_attention(q.contiguous(), a, 100))


def test_five_dimensions_are_four():
    from synthefy_nori_b200 import ops

    cache, g = make(6, 2, 300, 56)
    q = torch.randn(2, 50, 3, 2, 56, device="cuda", generator=g).to(torch.bfloat16)  # [b0, n, b1, heads, width]
    q5 = q.transpose(1, 2)
    o, lse = ops.block_cache_attention(q5, cache, 300, return_lse=True)
    o4, lse4 = ops.block_cache_attention(q5.reshape(6, 50, 2, 56), cache, 300, return_lse=True)
    assert o.shape == q5.shape and torch.equal(o.reshape(6, 50, 2, 56), o4) and torch.equal(lse, lse4)


def test_far_starts_and_shared_results_are_refused():
    from synthefy_nori_b200 import ops

    cache, g = make(2, 2, 200, 24)
    x = torch.randn(2, 10, 2, 24, device="cuda", generator=g).to(torch.bfloat16)
    before = [t.clone() for t in cache[:4]]
    for start in (2 ** 63 - 1, 2 ** 63 - 10, 2 ** 31, -(2 ** 63)):
        with pytest.raises(RuntimeError):
            ops.block_cache_write(cache, x, x, start=start)
        with pytest.raises((RuntimeError, ValueError, OverflowError, TypeError)):
            ops.block_cache_read(cache, start, start + 1)
    with pytest.raises(RuntimeError):
        ops.block_cache_attention(x, cache, 100, out=torch.empty(2, 1, 2, 24, device="cuda", dtype=x.dtype).expand_as(x))
    assert all(torch.equal(a, b) for a, b in zip(before, cache[:4]))


def test_device_starts_of_every_size():
    """Starts on the device below 0, over the end and at the ends of their type: rows outside are not written."""
    from synthefy_nori_b200 import ops

    starts = [-(2 ** 31), -5, 0, 250, 255, 256, 2 ** 31 - 1]
    cache = ops.block_cache(len(starts), 1, 256, 8)
    x = torch.arange(1, 11, device="cuda", dtype=torch.float32).view(1, 10, 1, 1).repeat(len(starts), 1, 1, 8)
    ops.block_cache_write(cache, x, x, start=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    k = values(cache)[0][:, 0, :, 0]
    for i, s in enumerate(starts):
        want = torch.zeros(256, dtype=torch.float64, device="cuda")
        for j in range(10):
            if 0 <= s + j < 256:
                want[s + j] = j + 1
        assert (k[i] - want).abs().max() <= 10 / 254 + 1e-6, s  # half a step


def test_two_captured_graphs_side_by_side():
    """Two graphs with workspaces of their own, replayed on two streams at once, again and again."""
    from synthefy_nori_b200 import ops

    cases = []
    for n, seed in ((1, 0), (200, 1)):
        cache, g = make(2, 2, 9000, 56, seed=seed)
        q = torch.randn(2, n, 2, 56, device="cuda", generator=g).to(torch.bfloat16)
        length = torch.full((2,), 9000, dtype=torch.int32, device="cuda")
        want = ops.block_cache_attention(q, cache, length)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = ops.block_cache_attention(q, cache, length)
        cases.append((graph, o, want, torch.cuda.Stream(), (cache, q, length)))  # (what a graph reads stays)
    for _ in range(20):
        for graph, o, _, s, _ in cases:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                o.zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, o, want, _, _ in cases:
        assert torch.equal(o, want)


def test_inference_mode_and_leaves():
    from synthefy_nori_b200 import ops

    with torch.inference_mode():
        cache, g = make(1, 2, 100, 16)
        q = torch.randn(1, 4, 2, 16, device="cuda", generator=g).to(torch.bfloat16)
        a = ops.block_cache_attention(q, cache, 100)
    cache, g = make(1, 2, 100, 16)
    q = torch.randn(1, 4, 2, 16, device="cuda", generator=g).to(torch.bfloat16).requires_grad_()
    b = ops.block_cache_attention(q, cache, 100)
    assert not b.requires_grad and torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 2, 130])
@pytest.mark.parametrize("dtype", ["block_int8", "block_fp8"])
def test_small_contexts_of_the_model(rows, dtype):
    """A context of one row and of one row more than a tile."""
    from synthefy_nori_b200.models.config import preset_config
    from synthefy_nori_b200.utils.loading import build_model

    torch.manual_seed(0)
    m = build_model(preset_config("nori-tiny")).to("cuda").eval()
    x = torch.randn(1, rows + 3, 5, device="cuda")
    y = x[..., 0]
    with torch.no_grad():
        a = m.apply_context_cache(x[:, rows:], m.build_context_cache(x[:, :rows], y[:, :rows]))
        b = m.apply_context_cache(x[:, rows:], m.build_context_cache(x[:, :rows], y[:, :rows], cache_dtype=dtype))
    assert torch.isfinite(b).all()
    assert torch.nn.functional.cosine_similarity(a.float().flatten(), b.float().flatten(), dim=0) > 0.998


@pytest.mark.parametrize("b,h,group,n,rows", [(19, 8, 1, 200, 3000), (25, 2, 3, 290, 1700), (5, 1, 1, 9000, 2000)])
@pytest.mark.parametrize("device_lengths", [False, True])
def test_more_work_than_one_wave(b, h, group, n, rows, device_lengths):
    """A little more work than there are SMs: some cells are taken whole, the keys of the last ones are split."""
    from synthefy_nori_b200 import ops

    cache, g = make(b, h, rows, 56, seed=b)
    q = torch.randn(b, n, h * group, 56, device="cuda", generator=g).to(torch.bfloat16)
    lengths = [rows - 100 * (i % 7) for i in range(b)] if device_lengths else [rows] * b
    given = torch.tensor(lengths, dtype=torch.int32, device="cuda") if device_lengths else rows
    o, lse = ops.block_cache_attention(q, cache, given, return_lse=True)
    check(q, cache, lengths, o, lse)


@pytest.mark.parametrize("b,h,n,rows", [(21, 8, 1024, 1000), (21, 8, 600, 130), (40, 8, 257, 700)])
def test_many_items_again_and_again(b, h, n, rows):
    """Short items in long rows of calls, a cold cache before some: every wait ends, every result is the first."""
    from synthefy_nori_b200 import ops

    cache, g = make(b, h, rows, 56, seed=n)
    q = (3 * torch.randn(b, n, h, 56, device="cuda", generator=g)).to(torch.bfloat16)
    first = ops.block_cache_attention(q, cache, rows)
    cold = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for i in range(400):
        if i % 8 == 0:
            cold.fill_(i & 255)
        o = ops.block_cache_attention(q, cache, rows)
        if i % 50 == 0:
            assert torch.equal(o, first)
    assert torch.equal(o, first)
    ops.check_status(q.device)


@pytest.mark.parametrize("n,group", [(257, 1), (100, 8), (33, 8)])
def test_captured_attention_write_attention(n, group):
    """Both kernels of a call and its joins, a write behind them and a second call, in one graph, replayed: what
    follows waits for all of them."""
    from synthefy_nori_b200 import ops

    cache, g = make(6, 2, 5000, 56, seed=n)
    q = torch.randn(6, n, 2 * group, 56, device="cuda", generator=g).to(torch.bfloat16)
    k, v = (torch.randn(6, 5000, 2, 56, device="cuda", generator=g) for _ in "kv")
    kept = [t.clone() for t in cache[:4]]

    def both():
        a = ops.block_cache_attention(q, cache, 5000)
        ops.block_cache_write(cache, k, v)
        return a, ops.block_cache_attention(q, cache, 5000)

    want = both()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for _ in range(5):
        for dst, src in zip(cache[:4], kept):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert not torch.equal(want[0], want[1])
