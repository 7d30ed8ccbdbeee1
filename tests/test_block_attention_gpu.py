"""Attention over a context cache in 8 bits with block scales, against the formula in 64 bits on the values
that the cache holds."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def values(cache):
    """(k, v) [batch, heads, capacity, D] in 64 bits."""
    out = []
    for code, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = code.float().double() * scale.double().repeat_interleave(cache.block, 2)[..., None]
        out.append(x[..., : cache.head_dim])
    return out


def reference(q, cache, lengths, scale=None):
    k, v = values(cache)
    b, n, hq, d = q.shape
    group = hq // k.shape[1]
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    s = torch.einsum("bnhd,bhmd->bhnm", q.double(), k) * (1 / math.sqrt(d) if scale is None else scale)
    off = torch.arange(k.shape[2], device=q.device) >= torch.as_tensor(lengths, device=q.device).view(-1, 1)
    s = s.masked_fill(off[:, None, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.masked_fill(lse == -math.inf, 0.0)[..., None])
    v = v.masked_fill(off[:, None, :, None], 0.0)
    # the size that roundings of the weights are relative to: sum of p |v|
    return torch.einsum("bhnm,bhmd->bnhd", p, v), lse, torch.einsum("bhnm,bhmd->bnhd", p, v.abs())


def check(q, cache, lengths, o, lse=None, scale=None):
    """Tolerances.  The result is rounded by half a step.  Weights are rounded to fp16 (2^-11) for the
    product, computed with 2^-17 or better (the polynomial 2^x 5e-6, sums in 32 bits), and scores in 32 bits carry
    (|q| . |k| scale) 2^-20: at most 2^-13 for scores up to 128 in magnitude.  Below 2^-14 fp16's values are
    2^-24 apart (its subnormals), so there half a step is 2^-25 whatever the value."""
    want, want_lse, size = reference(q, cache, lengths, scale)
    tol = want.abs() * torch.finfo(q.dtype).eps / 2 + size * (2.0 ** -11 + 2.0 ** -17 + 2.0 ** -13)
    tol += 2.0 ** -25 if q.dtype == torch.float16 else 1e-30
    err = (o.double() - want).abs()
    assert torch.isfinite(o).all() and (err <= tol).all(), float((err / tol).max())
    if lse is not None:
        assert lse.dtype == torch.float32 and torch.equal(lse == -math.inf, want_lse == -math.inf)
        fine = want_lse != -math.inf
        assert ((lse.double() - want_lse).abs()[fine] <= 2.0 ** -13 + 2.0 ** -23 * want_lse.abs()[fine]).all()


def make(batch, heads, rows, d, dtype=torch.int8, block=64, seed=0, spread=True):
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(seed)
    cache = ops.block_cache(batch, heads, rows, d, dtype=dtype, block=block)
    k, v = (torch.randn(batch, rows, heads, d, device="cuda", generator=g) for _ in "kv")
    if spread:  # scales that differ much from block to block
        size = torch.exp2(4 * torch.rand(1, rows, 1, 1, device="cuda", generator=g) - 3)
        step = torch.exp2(3 * torch.sin(torch.arange(rows, device="cuda") / 50.0)).view(1, rows, 1, 1)
        k, v = k * size, v * step
    ops.block_cache_write(cache, k, v)
    return cache, g


SIZES = [  # batch, kv heads, group, n, rows, d
    (1, 1, 1, 1, 1, 8), (2, 2, 1, 1, 31, 16), (1, 2, 1, 1, 33, 64), (3, 2, 1, 1, 1000, 56), (1, 1, 1, 1, 20000, 44),
    (2, 1, 8, 1, 777, 64), (2, 1, 8, 2, 129, 24), (1, 3, 1, 7, 400, 33), (1, 2, 1, 9, 400, 56), (2, 1, 3, 5, 640, 1),
    (2, 2, 1, 16, 300, 48), (1, 2, 1, 17, 300, 56), (1, 1, 2, 60, 130, 64), (2, 2, 1, 128, 128, 32), (1, 2, 1, 129, 257, 56),
    (1, 1, 1, 300, 1025, 64), (3, 1, 2, 200, 640, 44), (2, 8, 1, 257, 500, 56), (1, 1, 1, 1000, 3000, 13),
    (1, 1, 4, 100, 6001, 56), (40, 8, 1, 130, 200, 64),
]


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("qtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_attention_matches_formula(size, block, qtype, dtype):
    from synthefy_nori_b200 import ops

    b, h, group, n, rows, d = size
    cache, g = make(b, h, rows, d, dtype, block, seed=sum(size))
    q = (2 * torch.randn(b, n, h * group, d, device="cuda", generator=g)).to(qtype)
    o, lse = ops.block_cache_attention(q, cache, rows, return_lse=True)
    check(q, cache, [rows] * b, o, lse)


@pytest.mark.parametrize("n", [1, 12, 150])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_lengths_on_the_device(n, dtype):
    """Padded batches: empty sequences, single rows, lengths at, before and behind tiles and the capacity."""
    from synthefy_nori_b200 import ops

    lengths = [0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 640, 1000, 5, 0]
    cache, g = make(len(lengths), 2, 1000, 56, dtype, 32, seed=n)
    q = torch.randn(len(lengths), n, 2, 56, device="cuda", generator=g).to(torch.bfloat16)
    o, lse = ops.block_cache_attention(q, cache, torch.tensor(lengths, dtype=torch.int32, device="cuda"), return_lse=True)
    check(q, cache, lengths, o, lse)
    assert not o[0].any() and not o[-1].any()
    # taken into 0 .. capacity
    wild = torch.tensor([-5, 1 << 30] + lengths[2:], dtype=torch.int32, device="cuda")
    o2 = ops.block_cache_attention(q, cache, wild)
    check(q[1:2], type(cache)(*(t[1:2].contiguous() for t in cache[:4]), 56), [cache.capacity], o2[1:2])
    assert not o2[0].any() and torch.equal(o2[2:], o[2:])


@pytest.mark.parametrize("n", [1, 3, 40, 140])
def test_length_zero(n):
    from synthefy_nori_b200 import ops

    cache, g = make(2, 2, 128, 16)
    q = torch.randn(2, n, 2, 16, device="cuda").to(torch.float16)
    o, lse = ops.block_cache_attention(q, cache, 0, return_lse=True)
    assert not o.any() and (lse == -math.inf).all()


@pytest.mark.parametrize("d", [8, 20, 32, 40, 44, 56, 64])
@pytest.mark.parametrize("n", [1, 20, 260])
def test_rows_behind_the_length_do_not_count(n, d):
    """Whatever codes and scales lie behind the last row (NaN codes, infinities and NaN among the scales)."""
    from synthefy_nori_b200 import ops

    cache, g = make(2, 2, 512, d, torch.float8_e4m3fn, 32)
    q = torch.randn(2, n, 2, d, device="cuda", generator=g).to(torch.bfloat16)
    want = ops.block_cache_attention(q, cache, 161)
    for t in cache[:2]:
        behind = t.view(torch.int8)[:, :, 161:]
        behind.copy_(torch.randint(-128, 128, behind.shape, device="cuda"))
        behind[:, :, :3] = 127  # e4m3's NaN
    for t in cache[2:4]:
        t[:, :, 6:] = torch.tensor([math.nan, math.inf], device="cuda").repeat(5)
    assert torch.equal(ops.block_cache_attention(q, cache, 161), want)


@pytest.mark.parametrize("n", [1, 10, 130])
@pytest.mark.parametrize("which", ["q_nan", "q_inf", "k_nan", "v_nan"])
def test_non_finite_values_reach_their_rows_alone(n, which):
    from synthefy_nori_b200 import ops

    cache, g = make(2, 2, 300, 24)
    q = torch.randn(2, n, 2, 24, device="cuda", generator=g).to(torch.bfloat16)
    want = ops.block_cache_attention(q, cache, 300)
    hit = torch.zeros(2, n, 2, dtype=torch.bool, device="cuda")
    if which[0] == "q":
        q[1, n // 2, 1, 5] = math.nan if which == "q_nan" else -math.inf
        hit[1, n // 2, 1] = True
    else:
        (cache.k_scale if which[0] == "k" else cache.v_scale)[0, 1, 2] = math.nan
        hit[0, :, 1] = True
    o = ops.block_cache_attention(q, cache, 300)
    assert torch.equal(o.isnan().all(-1), hit) and torch.equal(o[~hit], want[~hit])


@pytest.mark.parametrize("n", [1, 140])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e4])
def test_magnitudes(n, size):
    """Queries and values far from 1: bf16's range, tiny and huge scales of K and V."""
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(1)
    cache = ops.block_cache(1, 2, 500, 32)
    k, v = (torch.randn(1, 500, 2, 32, device="cuda", generator=g) for _ in "kv")
    big = max(1e-9, 1 / size)
    ops.block_cache_write(cache, k * min(big, 1e6), v * size * 1e3)
    q = (torch.randn(1, n, 2, 32, device="cuda", generator=g) * size).to(torch.bfloat16)
    o, lse = ops.block_cache_attention(q, cache, 500, return_lse=True)
    check(q, cache, [500], o, lse)


@pytest.mark.parametrize("n", [1, 200])
def test_one_key_takes_all_or_a_million_share(n):
    """A peaked row, and many small weights behind one large: each below 2^-14 of it, together more."""
    from synthefy_nori_b200 import ops

    rows = 60000
    cache = ops.block_cache(1, 1, rows, 8)
    k = torch.zeros(1, rows, 1, 8, device="cuda")
    v = torch.ones(1, rows, 1, 8, device="cuda")
    k[0, 0, 0, 0] = 1.0
    v[0, 0] = -1.0
    ops.block_cache_write(cache, k, v)
    for gap in (5.0, 11.0, 14.0, 40.0):
        q = torch.zeros(1, n, 1, 8, device="cuda", dtype=torch.float16)
        q[..., 0] = gap
        o, lse = ops.block_cache_attention(q, cache, rows, scale=1.0, return_lse=True)
        check(q, cache, [rows], o, lse, scale=1.0)


@pytest.mark.parametrize("n", [1, 150])
def test_rising_scores_rescale(n):
    """Scores that rise from key to key: the running maximum moves all the way."""
    from synthefy_nori_b200 import ops

    rows = 1500
    cache = ops.block_cache(1, 2, rows, 8, block=32)
    k = torch.zeros(1, rows, 2, 8, device="cuda")
    k[0, :, 0, 0] = torch.linspace(0, 60, rows, device="cuda")
    k[0, :, 1, 0] = torch.linspace(60, 0, rows, device="cuda")
    v = torch.randn(1, rows, 2, 8, device="cuda")
    ops.block_cache_write(cache, k, v)
    q = torch.ones(1, n, 2, 8, device="cuda", dtype=torch.bfloat16)
    o, lse = ops.block_cache_attention(q, cache, rows, scale=1.5, return_lse=True)
    check(q, cache, [rows], o, lse, scale=1.5)


@pytest.mark.parametrize("n", [1, 5, 130])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_strided_queries_and_output(n, shift):
    """Token-major rows with two batch dimensions, at any alignment, written in place of other columns."""
    from synthefy_nori_b200 import ops

    B, T, H, D = 2, 3, 2, 24
    cache, g = make(B * T, H, 200, D)
    buf = torch.randn(B * n * T * 3 * H * D + 8, device="cuda", generator=g).to(torch.bfloat16)
    y = buf[shift:][: B * n * T * 3 * H * D].view(B, n, T, 3, H, D)
    q, out = (y[:, :, :, i].permute(0, 2, 1, 3, 4) for i in (0, 2))
    other = y[:, :, :, 1].clone()
    res, lse = ops.block_cache_attention(q, cache, 200, out=out, return_lse=True)
    assert res is out and torch.equal(y[:, :, :, 1], other) and lse.shape == (B * T, H, n)
    check(q.reshape(B * T, n, H, D), cache, [200] * 6, out.reshape(B * T, n, H, D), lse)


@pytest.mark.parametrize("n", [1, 30, 300])
def test_same_inputs_same_bits(n):
    from synthefy_nori_b200 import ops

    cache, g = make(3, 2, 3000, 56)
    q = torch.randn(3, n, 2, 56, device="cuda", generator=g).to(torch.bfloat16)
    first = ops.block_cache_attention(q, cache, 3000)
    assert all(torch.equal(ops.block_cache_attention(q, cache, 3000), first) for _ in range(5))


@pytest.mark.parametrize("n", [1, 257])
def test_new_contents_in_every_call(n):
    """Nothing of an earlier call is left to hide a read that comes too early: other data each time."""
    for seed in range(12):
        from synthefy_nori_b200 import ops

        cache, g = make(2, 8, 640, 64, seed=seed, spread=False)
        q = (2 * torch.randn(2, n, 8, 64, device="cuda", generator=g)).to(torch.float16)
        for _ in range(3):
            check(q, cache, [640] * 2, ops.block_cache_attention(q, cache, 640))


@pytest.mark.parametrize("n", [1, 200])
def test_captured_with_appends(n):
    """Append and attend in one graph, replayed as the cache grows; another graph shares nothing with it."""
    from synthefy_nori_b200 import ops

    cache, g = make(2, 2, 512, 32, block=32)
    q = torch.randn(2, n, 2, 32, device="cuda").to(torch.bfloat16)
    k, v = (torch.zeros(2, 1, 2, 32, device="cuda") for _ in "kv")
    pos = torch.full((2,), 300, dtype=torch.int32, device="cuda")

    def step():
        ops.block_cache_write(cache, k, v, start=pos)
        return ops.block_cache_attention(q, cache, pos + 1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = step()
        graphs.append((graph, o))
    for i in range(300, 330):
        x = torch.randn(2, 2, 1, 2, 32, device="cuda")
        k.copy_(x[0])
        v.copy_(x[1])
        pos.fill_(i)
        graph, o = graphs[i % 2]
        graph.replay()
        check(q, cache, [i + 1] * 2, o)


@pytest.mark.parametrize("n", [1, 200])
def test_streams_side_by_side(n):
    """Calls on several streams at once, each with its own inputs."""
    from synthefy_nori_b200 import ops

    work = []
    for i in range(4):
        cache, g = make(2, 2, 2000 + 100 * i, 56, seed=i)
        q = torch.randn(2, n, 2, 56, device="cuda", generator=g).to(torch.bfloat16)
        work.append((q, cache, 2000 + 100 * i, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for q, cache, rows, stream in work:
            with torch.cuda.stream(stream):
                outs.append((q, cache, rows, ops.block_cache_attention(q, cache, rows)))
    torch.cuda.synchronize()
    for q, cache, rows, o in outs:
        check(q, cache, [rows] * 2, o)


def test_far_offsets():
    """A cache of more than 2^31 bytes: the last sequence's rows."""
    from synthefy_nori_b200 import ops

    cache = ops.block_cache(3, 1, 20_000_000, 56)
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(3, 3000, 1, 56, device="cuda", generator=g) for _ in "kv")
    ops.block_cache_write(cache, k, v, start=20_000_000 - 3000)
    ko, _ = ops.block_cache_read(cache, 20_000_000 - 3000, 20_000_000, dtype=torch.float32)
    assert ((ko - k).abs() <= k.abs().amax() / 254 + 1e-6).all()
    # every row before is zero: scores 0, values 0
    q = (30 * torch.randn(3, 2, 1, 56, device="cuda", generator=g)).to(torch.bfloat16)
    o, lse = ops.block_cache_attention(q, cache, 20_000_000, return_lse=True)
    s = torch.einsum("bnhd,bmhd->bhnm", q.double(), ko.double()) / math.sqrt(56)
    want_lse = torch.logsumexp(torch.cat((s, torch.full((3, 1, 2, 1), math.log(20_000_000 - 3000), device="cuda",
                                                       dtype=torch.float64)), 3), 3)
    # 2^-13 as in check(), and 2e7 weights added in 32 bits in runs of at most 2^10: 2^-24 for each addition
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -13 + 2.0 ** -14).all()


def test_write_read_attend_together():
    """A context written in chunks, read back for a plain attention, and attended to directly: the same result."""
    from synthefy_nori_b200 import ops

    g = torch.Generator(device="cuda").manual_seed(2)
    B, N, H, D = 3, 1000, 2, 56
    k, v = (torch.randn(B, N, H, D, device="cuda", generator=g).to(torch.bfloat16) for _ in "kv")
    q = torch.randn(B, 33, H, D, device="cuda", generator=g).to(torch.bfloat16)
    for dtype in ops.BLOCK_CACHE_TYPES:
        cache = ops.block_cache(B, H, N, D, dtype=dtype, block=64)
        for at in range(0, N, 192):  # chunks of whole blocks: the codes of a single write
            ops.block_cache_write(cache, k[:, at : at + 192], v[:, at : at + 192], start=at)
        once = ops.block_cache(B, H, N, D, dtype=dtype, block=64)
        ops.block_cache_write(once, k, v)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache[:4], once[:4]))
        kb, vb = ops.block_cache_read(cache, 0, N, dtype=torch.float32)
        s = torch.einsum("bnhd,bmhd->bhnm", q.double(), kb.double()) / math.sqrt(D)
        want = torch.einsum("bhnm,bmhd->bnhd", torch.softmax(s, -1), vb.double())
        o = ops.block_cache_attention(q, cache, N)
        assert ((o.double() - want).abs() <= want.abs() * 2.0 ** -8 + vb.abs().max() * 2.0 ** -10).all()
