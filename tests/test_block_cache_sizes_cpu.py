"""Sizes of a block-scaled cache are whole numbers."""

import numpy as np
import pytest

from synthefy_nori_b200 import ops


@pytest.mark.parametrize("kw", [dict(capacity=100.5), dict(head_dim=16.5), dict(batch=1.5), dict(heads=2.0), dict(block=64.0)])
def test_fractions_are_refused(kw):
    args = dict(batch=2, heads=2, capacity=100, head_dim=16, block=64) | kw
    with pytest.raises((TypeError, ValueError)):
        ops.block_cache(**args, device="cpu")


def test_whole_numbers_of_numpy():
    c = ops.block_cache(*(np.int64(x) for x in (2, 3, 100, 20)), device="cpu")
    assert c.k.shape == (2, 3, 128, 24) and c.head_dim == 20 and type(c.head_dim) is int
