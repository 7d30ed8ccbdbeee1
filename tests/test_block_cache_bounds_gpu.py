"""How far values move that are appended row by row, and the forms of the attention that only long contexts reach."""

import math

import pytest
import torch

from test_block_attention_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("block", [32, 64, 128])
@pytest.mark.parametrize("growth", [1.0, 1.03, 1.5])
def test_appended_rows_stay_near_what_was_given(dtype, block, growth):
    """A row is rounded as it is written and once more each time its block's scale grows.  int8: half a step of the
    scale then.  e4m3: half a step of the value, 2^-4 of it, or 2^-10 of the scale among its subnormals.  (Scales and
    products are rounded to fp32: 2^-22 of a value's largest code.)"""
    from synthefy_nori_b200 import ops

    n, top = 2 * block + 5, 127.0 if dtype == torch.int8 else 448.0
    g = torch.Generator(device="cuda").manual_seed(block)
    size = growth ** torch.arange(n, device="cuda", dtype=torch.float64) if growth < 1.5 else 1.0 + torch.arange(
        n, device="cuda", dtype=torch.float64) % 7 * 2
    x = (torch.randn(1, n, 2, 24, device="cuda", generator=g).double() * size.view(1, -1, 1, 1)).float()
    cache = ops.block_cache(1, 2, n, 24, dtype=dtype, block=block)
    bound = torch.zeros(n, 2, 24, dtype=torch.float64, device="cuda")
    was = torch.zeros(2, dtype=torch.float64, device="cuda")
    growths = 0
    for i in range(n):
        ops.block_cache_write(cache, x[:, i : i + 1], x[:, i : i + 1], start=i)
        b = i // block
        s = cache.k_scale[0, :, b].double()
        if i % block == 0:
            was = torch.zeros_like(s)
        grew = s > was
        growths += int(grew.sum()) if i % block else 0
        rows = torch.arange(b * block, i + 1, device="cuda")
        again = torch.where(rows[:, None, None] == i, True, grew[None, :, None])  # the new row, and all where it grew
        now = x[0, rows].double().abs() + bound[rows]
        step = s[None, :, None] * (0.5 if dtype == torch.int8 else 2.0 ** -10) + s[None, :, None] * top * 2.0 ** -22
        if dtype != torch.int8:
            step = step + now * 2.0 ** -4
        bound[rows] += torch.where(again, step, 0.0)
        was = s
    k, v = ops.block_cache_read(cache, 0, n, dtype=torch.float32)
    for got in (k, v):
        assert ((got[0].double() - x[0].double()).abs() <= bound).all()
    assert growths > (3 if growth == 1.0 else 10)


@pytest.mark.parametrize("n", [1, 12])
@pytest.mark.parametrize("device_lengths", [False, True])
def test_parts_beyond_thirty_two(n, device_lengths):
    """One row tile against 100,003 keys: the keys are split 384 times, and 48 parts joined."""
    from synthefy_nori_b200 import ops

    rows = 100_003
    cache, g = make(1, 1, rows, 56, seed=n)
    q = (2 * torch.randn(1, n, 1, 56, device="cuda", generator=g)).to(torch.bfloat16)
    for length in (rows, 90_001, 1):
        given = torch.tensor([length], dtype=torch.int32, device="cuda") if device_lengths else length
        o, lse = ops.block_cache_attention(q, cache, given, return_lse=True)
        check(q, cache, [length], o, lse)


@pytest.mark.parametrize("n", [2, 40, 300])
@pytest.mark.parametrize("size", [1.0, 30.0])
def test_results_far_into_a_long_cache(n, size):
    """A cache of more than 2^31 bytes whose last 3000 rows alone were written: zeros elsewhere, with scores 0."""
    from synthefy_nori_b200 import ops

    rows, last = 20_000_000, 3000
    cache = ops.block_cache(3, 1, rows, 56)
    g = torch.Generator(device="cuda").manual_seed(n)
    k, v = (torch.randn(3, last, 1, 56, device="cuda", generator=g) for _ in "kv")
    ops.block_cache_write(cache, k, v, start=rows - last)
    k, v = (t.double() for t in ops.block_cache_read(cache, rows - last, rows, dtype=torch.float32))
    q = (size * torch.randn(3, n, 1, 56, device="cuda", generator=g)).to(torch.bfloat16)
    o, lse = ops.block_cache_attention(q, cache, rows, return_lse=True)
    s = torch.einsum("bnhd,bmhd->bhnm", q.double(), k) / math.sqrt(56)
    zeros = torch.full((3, 1, n, 1), math.log(rows - last), device="cuda", dtype=torch.float64)
    want_lse = torch.logsumexp(torch.cat((s, zeros), 3), 3)
    p = torch.exp(s - want_lse[..., None])
    want, near = torch.einsum("bhnm,bmhd->bnhd", p, v), torch.einsum("bhnm,bmhd->bnhd", p, v.abs())
    # 2e7 weights added in 32 bits in runs of at most 2^10: 2^-14 of the sum; weights as fp16 2^-11; scores of up to
    # 64 |size| / 8 with 2^-20 of |q| |k| each: 2^-11; the result half a step.  And where a column of the largest weight's
    # key holds code 0, the others count alone: fp16's values are 2^-24 apart below 2^-14, half of that is 2^-32 of the
    # largest weight (which is 2^7 or more), and so much of the largest value, for each key.
    assert ((lse.double() - want_lse).abs() <= 2.0 ** -11 + 2.0 ** -14).all()
    tol = want.abs() * 2.0 ** -8 + near * (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -14 + 2.0 ** -17)
    tol += last * v.abs().max() * 2.0 ** -32
    assert ((o.double() - want).abs() <= tol).all()
