"""Arguments of the block-scaled cache that are refused on the host: memory that is read and written in one call, and
numbers that are no whole numbers."""

import pytest
import torch

from test_block_attention_gpu import check, make

pytestmark = pytest.mark.gpu


def _refused(*calls):
    for call in calls:
        with pytest.raises((RuntimeError, ValueError, TypeError)):
            call()


@pytest.mark.parametrize("n", [1, 40, 300])
def test_out_that_shares_memory(n):
    """With q (all of it, a column, a row further on), with the cache, with the lengths, and with itself; columns of one
    buffer side by side are taken."""
    from synthefy_nori_b200 import ops

    H, D = 2, 24
    cache, g = make(2, H, 256, D)
    buf = torch.randn(2 * (n + 1), 4 * H * D, device="cuda", generator=g).to(torch.bfloat16)
    y = buf.view(2, n + 1, 4, H, D)
    q = y[:, :n, 0]
    flat = buf.view(-1)
    shifted = flat[D // 2 :].as_strided(q.shape, q.stride(), flat.storage_offset() + D // 2)
    in_cache = cache.k.view(-1).view(torch.bfloat16)
    before = [t.clone() for t in (buf, *cache[:4])]
    for lengths in (200, torch.full((2,), 200, dtype=torch.int32, device="cuda")):
        _refused(
            lambda: ops.block_cache_attention(q, cache, lengths, out=q),
            lambda: ops.block_cache_attention(q, cache, lengths, out=y[:, 1:, 0]) if n > 1 else ops.block_cache_attention(
                q, cache, lengths, out=q),
            lambda: ops.block_cache_attention(q, cache, lengths, out=shifted),
            lambda: ops.block_cache_attention(q[:, :1], cache, lengths, out=in_cache[: 2 * H * D].view(2, 1, H, D)),
            lambda: ops.block_cache_attention(q[:, :1], cache, lengths, out=cache.v_scale.view(-1).view(torch.bfloat16)[
                : 1].as_strided((2, 1, H, D), (0, 0, 0, 1))),
            # rows that follow one another at less than a row's length
            lambda: ops.block_cache_attention(q, cache, lengths, out=flat.as_strided(
                q.shape, ((n + 1) * H * D, H * D - 8, D, 1), 0)) if n > 1 else ops.block_cache_attention(q, cache, lengths, out=q),
        )
    words = torch.full((2 * n * H * D,), 200, dtype=torch.int32, device="cuda")
    _refused(lambda: ops.block_cache_attention(q, cache, words[:2], out=words.view(torch.bfloat16)[: q.numel()].view(q.shape)))
    assert all(torch.equal(a, b) for a, b in zip(before, (buf, *cache[:4])))
    out = y[:, :n, 3]
    check(q, cache, [200, 200], ops.block_cache_attention(q, cache, 200, out=out))


def test_writes_that_share_memory():
    """K and V of one memory, scales of one memory, and rows that lie in the cache itself."""
    from synthefy_nori_b200 import ops

    c = ops.block_cache(1, 2, 256, 16)
    x = torch.ones(1, 10, 2, 16, device="cuda")
    before = [t.clone() for t in c[:4]]
    inside = c.k.view(-1).view(torch.float32)[: 10 * 32].view(1, 10, 2, 16)
    _refused(
        lambda: ops.block_cache_write(ops.BlockCache(c.k, c.k, c.k_scale, c.v_scale, 16), x, x),
        lambda: ops.block_cache_write(ops.BlockCache(c.k, c.v, c.k_scale, c.k_scale, 16), x, x),
        lambda: ops.block_cache_write(c, inside, x), lambda: ops.block_cache_write(c, x, inside),
    )
    assert all(torch.equal(a, b) for a, b in zip(before, c[:4]))
    ops.block_cache_write(c, x, x)  # (one tensor for keys and values)
    # a cache whose keys are its values can be read
    same = ops.BlockCache(c.k, c.k, c.k_scale, c.k_scale, 16)
    q = torch.ones(1, 1, 2, 16, device="cuda", dtype=torch.bfloat16)
    assert (ops.block_cache_attention(q, same, 10) == 1).all()


def test_lengths_and_places_are_whole_numbers():
    """A fraction is refused, not cut off; numpy's whole numbers are taken."""
    import numpy as np

    from synthefy_nori_b200 import ops

    c, g = make(1, 2, 200, 16)
    x = torch.randn(1, 10, 2, 16, device="cuda", generator=g)
    q = x.bfloat16()
    before = [t.clone() for t in c[:4]]
    _refused(
        lambda: ops.block_cache_attention(q, c, 10.9), lambda: ops.block_cache_attention(q, c, "10"),
        lambda: ops.block_cache_attention(q, c, np.float64(10.0)), lambda: ops.block_cache_write(c, x, x, start=0.5),
        lambda: ops.block_cache_read(c, 0.5, 10), lambda: ops.block_cache_read(c, 0, 9.5),
    )
    assert all(torch.equal(a, b) for a, b in zip(before, c[:4]))
    assert torch.equal(ops.block_cache_attention(q, c, np.int64(10)), ops.block_cache_attention(q, c, 10))
