"""LayerNorm over the last dimension on the native kernels, with its gradients.

``layer_norm`` is the autograd form; ``layer_norm_fwd`` / ``layer_norm_bwd`` are the two
kernels for autograd nodes that keep their own saved tensors.  Statistics and sums are fp32;
the weight's and bias's gradients are added in a fixed order (the same inputs give the same
bits).
"""

from __future__ import annotations

import torch

from synthefy_nori_b200.ops.api import _lib

__all__ = ["layer_norm", "layer_norm_fwd", "layer_norm_bwd"]

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t [..., C]`` as [R, C] with contiguous columns (a view where the strides allow it)."""
    if t.dim() == 2 and t.stride(1) == 1 and t.shape[1] and t.stride(0) >= 0:
        return t
    if t.dim() == 0:
        raise ValueError("layer_norm: at least one dimension expected")
    t = t.reshape(-1, t.shape[-1]) if t.shape[-1] else t.reshape(0, 0)
    ok = t.shape[-1] <= 1 or (t.stride(1) == 1 and t.stride(0) >= 0)
    return t if ok else t.contiguous()


def _check(x: torch.Tensor, out_dtype) -> bool:
    if not x.is_cuda:
        raise ValueError("layer_norm: a CUDA tensor expected")
    if x.dtype not in _FLOATS:
        raise ValueError(f"layer_norm: fp32, bf16 or fp16 expected, got {x.dtype}")
    if out_dtype not in (None, x.dtype, torch.float32):
        raise ValueError(f"layer_norm: out_dtype must be x's type or fp32, got {out_dtype}")
    return out_dtype == torch.float32


def layer_norm_fwd(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, out_dtype=None):
    """``(y, mean, rstd)`` of ``x [..., C]`` (fp32, bf16 or fp16; ``y`` in x's type or, with
    ``out_dtype``, fp32); ``mean`` and ``rstd`` are fp32, one per row."""
    f32 = _check(x, out_dtype)
    y, mean, rstd = _lib().layer_norm_fwd(_rows(x), weight, bias, eps, f32)
    return y if x.dim() == 2 else y.view(x.shape), mean, rstd


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight=None, *,
                   weight_grad: bool | None = None, bias_grad: bool = True):
    """``(dx, dw, db)`` for ``dy`` of x's type or fp32; ``dw`` (wanted by default where there
    is a weight) and ``db`` are fp32 ``[C]``, or None where unwanted."""
    _check(x, None)
    weight_grad = weight is not None if weight_grad is None else weight_grad
    dx, dw, db = _lib().layer_norm_bwd(_rows(dy), _rows(x), mean, rstd, weight, bool(weight_grad), bool(bias_grad))
    return dx if x.dim() == 2 else dx.view(x.shape), dw if weight_grad else None, db if bias_grad else None


def layer_norm(x: torch.Tensor, weight=None, bias=None, eps: float = 1e-5, out_dtype=None) -> torch.Tensor:
    """LayerNorm of ``x [..., C]`` over its last dimension, differentiable in ``x``, ``weight``
    and ``bias`` (``[C]`` or None, any floating type on x's device; fp32 and x's type are read as
    they are, others cast).  The result has x's type,
    or fp32 with ``out_dtype=torch.float32``."""
    f32 = _check(x, out_dtype)
    if x.dim() == 0:
        raise ValueError("layer_norm: at least one dimension expected")
    return _lib().layer_norm(x, weight, bias, eps, f32, torch.autograd.forward_ad._current_level >= 0)
