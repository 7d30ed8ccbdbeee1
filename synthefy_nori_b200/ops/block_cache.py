"""Context cache in 8 bits with a scale for each block of rows and head, and the attention that reads it.

A ``BlockCache`` holds keys and values as int8 or e4m3 codes ``[batch, heads, capacity, W]`` (``W`` the
head width up to a multiple of 8) with one fp32 scale per (sequence, head, block of 32, 64 or 128
rows); a value is code * scale.  ``block_cache_write`` quantises rows as they are written, at the end of
what a sequence holds (rows behind them in the same block keep their codes and get the block's new scale,
so rows in the middle are rewritten by whole blocks); ``block_cache_read`` gives them back; ``block_cache_attention`` runs
query rows against the codes themselves (any number of rows, a single one included; shared K/V
heads).  Against one scale per (row, head) vector (``quantize_int8``) the scales take 4 / (block D)
instead of 4 / D of the codes, and the attention needs no bf16 copy of the cache.

Everything runs on the current stream of the cache's device and can be captured into a CUDA graph;
``start``, ``counts`` and ``lengths`` may be int32 tensors on the device, read when the kernel runs.  No
operation has a gradient: results have no graph.
"""

from __future__ import annotations

from operator import index
from typing import NamedTuple

import torch

from synthefy_nori_b200.ops.api import _lib, status_word

__all__ = ["BlockCache", "block_cache", "block_cache_write", "block_cache_read", "block_cache_attention",
           "BLOCK_CACHE_TYPES"]

#: Types of the stored codes.
BLOCK_CACHE_TYPES = (torch.int8, torch.float8_e4m3fn)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_ROWS = 128  # the capacity is a multiple


class BlockCache(NamedTuple):
    """Codes ``k``, ``v`` [batch, heads, capacity, W], scales [batch, heads, capacity / block] (fp32),
    and the head width."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    head_dim: int

    @property
    def block(self) -> int:
        return self.k.shape[2] // self.k_scale.shape[2]

    @property
    def capacity(self) -> int:
        return self.k.shape[2]

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in self[:4])


def block_cache(batch: int, heads: int, capacity: int, head_dim: int, *, dtype=torch.int8, block: int = 64,
                device="cuda") -> BlockCache:
    """An empty cache (zeros) for ``capacity`` rows of ``batch`` sequences (made a multiple of 128)."""
    if dtype not in BLOCK_CACHE_TYPES:
        raise ValueError(f"block_cache: int8 or float8_e4m3fn expected, got {dtype}")
    batch, heads, capacity, head_dim, block = (index(x) for x in (batch, heads, capacity, head_dim, block))
    if block not in (32, 64, 128):
        raise ValueError(f"block_cache: blocks of 32, 64 or 128 rows expected, got {block}")
    if not 1 <= head_dim <= 64:
        raise ValueError(f"block_cache: head widths of 1 to 64 expected, got {head_dim}")
    if batch < 0 or heads < 0 or capacity < 0:
        raise ValueError("block_cache: negative size")
    cap = max(_ROWS, -(-capacity // _ROWS) * _ROWS)
    width = -(-head_dim // 8) * 8
    k, v = (torch.zeros(batch, heads, cap, width, dtype=dtype, device=device) for _ in "kv")
    ks, vs = (torch.zeros(batch, heads, cap // block, dtype=torch.float32, device=device) for _ in "kv")
    return BlockCache(k, v, ks, vs, head_dim)


def _cuda(t, who: str, what: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{who}: {what} must be a CUDA tensor")


def _int_or_tensor(x):
    """(value, device tensor or None) of an int or an int32 tensor."""
    if isinstance(x, torch.Tensor):
        return 0, x
    return index(x), None


def block_cache_write(cache: BlockCache, k: torch.Tensor, v: torch.Tensor, start=0, counts=None) -> None:
    """Quantises ``k``, ``v`` [batch, n, heads, head_dim] (or two batch dimensions; fp32, bf16 or fp16,
    any strides with contiguous columns) into rows ``start .. start + n`` of each sequence.

    ``start`` is an int or int32 [batch] on the device, ``counts`` (int32 [batch], default n) how many
    of the n rows of a sequence are there.  ``k`` and ``v`` share no memory with the cache.  A block's scale is its largest magnitude over 127 (int8)
    or 448 (e4m3).  Where earlier rows of the first block stay (``start`` inside a block), its scale
    only grows, and they are quantised again under it when it does: each growth rounds them once more (half a
    step of the new scale in int8, up to 2^-4 of the value in e4m3), up to block - 1 times where rows come one
    by one.  Rows written by whole blocks are rounded once.  Rows
    at or behind ``start + counts`` in the last block end there: their codes stay, but under its new scale.
    With device values, rows outside the capacity are not written.  A block that gets an infinity or
    a NaN reads as NaN."""
    _cuda(cache.k, "block_cache_write", "the cache")
    _cuda(k, "block_cache_write", "k")
    _cuda(v, "block_cache_write", "v")
    at, at_dev = _int_or_tensor(start)
    _lib().block_cache_write(*cache[:4], cache.head_dim, k, v, at, at_dev, counts)
    torch.autograd.graph.increment_version(list(cache[:4]))


def block_cache_read(cache: BlockCache, start: int = 0, end: int | None = None, dtype=torch.bfloat16):
    """``(k, v)`` [batch, end - start, heads, head_dim] of rows ``start .. end`` (default: the capacity) as
    fp32, bf16 or fp16: code * scale, rounded once.  (A view of head-major memory.)"""
    _cuda(cache.k, "block_cache_read", "the cache")
    if dtype not in _FLOATS:
        raise ValueError(f"block_cache_read: fp32, bf16 or fp16 expected, got {dtype}")
    start, end = index(start), cache.capacity if end is None else index(end)
    k, v = _lib().block_cache_read(*cache[:4], cache.head_dim, start, end - start, dtype)
    return k, v


def block_cache_attention(q: torch.Tensor, cache: BlockCache, lengths, *, scale: float | None = None,
                          return_lse: bool = False, out: torch.Tensor | None = None):
    """``softmax(scale q K^T) V`` over the first ``lengths`` rows of each sequence (an int, or int32 [batch]
    on the device, taken into 0 .. capacity), in q's type.

    ``q`` is bf16 or fp16 [batch, n, heads, head_dim] (or two batch dimensions) with any strides and
    contiguous columns; its heads are a multiple of the cache's, neighbours sharing a K/V head.
    ``scale`` (default head_dim ** -0.5) is positive.  ``out``, if given, has q's shape and type and shares
    no memory with q, the cache or the lengths (columns of one buffer side by side share none).  With ``return_lse`` also the natural log-sum-exp, fp32 [batch, heads, n].
    Length 0 gives zeros and -inf; a query row with an infinity or a NaN, or scores past fp32's range, give NaN.

    Sums, maxima and results are held in fp32; weights are rounded to fp16 for the product with V, relative to the
    largest weight times its block's scale of V (11 bits down to 2^-21 of that, 2^-32 of it below).  A block's scale of V counts as
    2^-80 and as 2^-100 of the largest at least: the result is off by 2^-100 of the largest value of V at most, the
    log-sum-exp not at all.  Where keys are split over SMs, partial results take up to 160 MB while a call runs.
    After a wait on the device has run out (``ops.check_status`` raises) rows may not have been written."""
    k = cache.k
    if not k.is_cuda or not isinstance(q, torch.Tensor) or not q.is_cuda:
        raise ValueError("block_cache_attention: q and the cache must be CUDA tensors")
    if out is not None and not (isinstance(out, torch.Tensor) and out.shape == q.shape and out.dtype == q.dtype
                                and out.device == q.device):
        raise ValueError("block_cache_attention: out must have q's shape, type and device")
    length, length_dev = _int_or_tensor(lengths)
    res, lse = _lib().block_cache_attention(q, k, cache.v, cache.k_scale, cache.v_scale, cache.head_dim, length, length_dev,
                                            cache.head_dim ** -0.5 if scale is None else scale, out, return_lse,
                                            status_word(k.device))
    if out is not None:
        torch.autograd.graph.increment_version(out)
        res = out
    return (res, lse) if return_lse else res
