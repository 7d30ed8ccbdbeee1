"""Whether two strided views reach the same memory, against every address written out."""

import random

import pytest
import torch

from synthefy_nori_b200 import ops

pytestmark = pytest.mark.skipif(not ops.native_available(), reason="the extension is not built")


def _bytes(t):
    """Addresses of the first byte of every element."""
    at = torch.zeros(1, dtype=torch.int64)
    for n, s in zip(t.shape, t.stride()):
        at = (at[:, None] + torch.arange(n) * s).reshape(-1)
    return (at * t.element_size() + t.data_ptr()).tolist()


def _reach(t):
    return {p + i for p in _bytes(t) for i in range(t.element_size())}


@pytest.mark.parametrize("seed", range(100))
def test_any_two_views(seed):
    r = random.Random(seed)
    buf = torch.zeros(16384, dtype=torch.uint8)
    views = []
    for _ in "ab":
        t = buf[r.choice([0, 0, 4, 64, 132]):]
        t = t[: t.numel() // 4 * 4].view(r.choice([torch.int16, torch.float32, torch.uint8]))
        sizes = [r.choice([1, 2, 3, 5]) for _ in range(r.randint(1, 4))]
        strides = [r.choice([0, 1, 2, 3, 4, 8, 16, 24, 48]) for _ in sizes]
        views.append(t.as_strided(sizes, strides, t.storage_offset() + r.randint(0, 40)))
    a, b = views
    assert ops.lib().shares_memory(a, b) == bool(_reach(a) & _reach(b))
    at = _bytes(a)
    assert ops.lib().shares_memory(a) == (len(_reach(a)) < len(at) * a.element_size())


def test_views_of_one_buffer():
    """Columns side by side share nothing; one column or one row more does."""
    y = torch.zeros(2, 50, 3, 3, 2, 24, dtype=torch.bfloat16)
    shares = ops.lib().shares_memory
    q, k, v = (y[:, :, :, i].permute(0, 2, 1, 3, 4) for i in range(3))
    assert not shares(q, v) and not shares(q, k) and shares(q, q) and not shares(q)
    w = y.view(2, 50, 3, 144)
    assert shares(w[..., :49], w[..., 48:96]) and not shares(w[..., :48], w[..., 48:96])
    assert shares(w[:, :26], w[:, 25:]) and not shares(w[:, :25], w[:, 25:])
    assert shares(w[:, :, :1].expand(-1, -1, 3, -1), w) and shares(w[:, :, :1].expand(-1, -1, 3, -1))
    assert not shares(w[:0], w) and not shares(torch.zeros(5), torch.zeros(5))
    big = torch.zeros(1, dtype=torch.bfloat16).expand(1 << 20, 1 << 20)
    assert shares(big) and shares(big, big)
