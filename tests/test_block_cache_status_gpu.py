"""What block-scaled attention does once a wait on the device has run out (the status word says so)."""

import pytest
import torch

from test_block_attention_gpu import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,rows", [(200, 100), (1100, 128)])
def test_after_a_timeout_many_rows_are_left_alone(n, rows):
    """Whole CTAs leave, their tensor memory freed: nothing is written, and calls work again once the word is cleared."""
    from synthefy_nori_b200 import ops

    cache, g = make(3, 4, rows, 56)
    q = torch.randn(3, n, 4, 56, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    word = ops.status_word(q.device)
    try:
        word.fill_(2)
        for _ in range(3):
            ops.block_cache_attention(q, cache, rows, out=out)
        with pytest.raises(RuntimeError, match="timeout"):
            ops.check_status(q.device)
    finally:
        word.zero_()
    assert (out == 7.0).all()
    for _ in range(3):
        check(q, cache, [rows] * 3, ops.block_cache_attention(q, cache, rows, out=out))
    ops.check_status(q.device)


@pytest.mark.parametrize("n,rows", [(200, 700), (1100, 3000), (1, 100003)])
def test_after_a_timeout_no_parts_are_joined(n, rows):
    """Where the keys are split, the join does not read parts that were never written."""
    from synthefy_nori_b200 import ops

    cache, g = make(1, 2, rows, 56)
    q = torch.randn(1, n, 2, 56, device="cuda", generator=g).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    word = ops.status_word(q.device)
    try:
        word.fill_(2)
        for _ in range(3):
            ops.block_cache_attention(q, cache, rows, out=out)
    finally:
        word.zero_()
    assert (out == 7.0).all()
    check(q, cache, [rows], ops.block_cache_attention(q, cache, rows, out=out))
