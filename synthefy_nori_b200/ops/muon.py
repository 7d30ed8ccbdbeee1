"""Muon on the native kernels: orthogonalisation by Newton-Schulz products and the whole
optimizer step for a set of matrices in flat buffers.

``newton_schulz`` replaces a matrix by an approximation of its orthogonal polar factor:
``X <- a X + (b A + c A^2) X`` with ``A = X X^T``, from ``X = G / (|G|_F + eps)``.  The
products run on tcgen05 with fp16 operands and fp32 accumulation while the iterate keeps 22
or more bits, so five steps are within 3e-3 (2-norm) of the exact iteration whatever the
spectrum of ``G`` (1e-5 for up to 32 columns, or rows, and 1,536 of the other): a bf16 result
carries all of it.  The iterate's scale follows the result, so more steps add their own error
alone: 1e-2 after 64 on most matrices with the coefficients below (one whose singular values pass
the iteration's repelling fixed point, 0.868, spreads roundings as any precision does), 1.5e-3
after 64 of a convergent iteration.

After a bounded wait of any native kernel on the device has run out (``ops.check_status``
raises), ``muon_step`` leaves its buffers as they are and ``newton_schulz`` its output
unwritten; a wait of their own that runs out leaves results incomplete.

``MuonPlan`` describes which ranges of a flat parameter buffer are matrices; ``muon_step``
runs clipping, momentum, orthogonalisation, weight decay, update and parameter average on
all of them.
"""

from __future__ import annotations

import torch

from synthefy_nori_b200.ops.api import _lib, status_word

__all__ = ["newton_schulz", "MuonPlan", "muon_step", "NS_COEFFS"]

#: The quintic iteration's coefficients (K. Jordan et al., 2024).
NS_COEFFS = (3.4445, -4.7750, 2.0315)
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_ADJUST = {"match_rms_adamw": 0, "original": 1, "nd": 2}


def newton_schulz(g: torch.Tensor, steps: int = 5, eps: float = 1e-7, coeffs=NS_COEFFS, out_dtype=None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of every matrix of ``g [..., rows, cols]`` (fp32, bf16
    or fp16; any strides), in ``out_dtype`` (default: g's; about 11 significant bits are
    right).  ``out``, if given, is contiguous, of g's shape, and sets the type; it may be
    ``g`` itself, but share no other memory with it.  A matrix of zeros gives zeros; a NaN or an infinity makes its own matrix
    NaN and no other.  ``steps`` is 1 to 64, the first coefficient 1 to 1024; the coefficients
    are such that the iteration stays bounded (singular values of 100 leave fp16's range).  Not differentiable: the result has no graph."""
    if not isinstance(g, torch.Tensor) or not g.is_cuda:
        raise ValueError("newton_schulz: a CUDA tensor expected")
    if g.dim() < 2:
        raise ValueError("newton_schulz: a matrix or a batch of matrices [..., rows, cols] expected")
    if g.dtype not in _FLOATS:
        raise ValueError(f"newton_schulz: fp32, bf16 or fp16 expected, got {g.dtype}")
    if out_dtype is not None and out_dtype not in _FLOATS:
        raise ValueError(f"newton_schulz: out_dtype must be fp32, bf16 or fp16, got {out_dtype}")
    if out is not None:
        if out.shape != g.shape or out.device != g.device or not out.is_contiguous() or out.dtype not in _FLOATS:
            raise ValueError("newton_schulz: out must be contiguous fp32, bf16 or fp16, of g's shape and on its device")
        if out_dtype is not None and out.dtype != out_dtype:
            raise ValueError(f"newton_schulz: out is {out.dtype}, out_dtype {out_dtype}")
    res = _lib().newton_schulz(g if g.is_contiguous() else g.contiguous(), out, out_dtype, steps, eps, coeffs,
                               status_word(g.device))
    if out is None:
        return res
    torch.autograd.graph.increment_version(out)
    return out


class MuonPlan:
    """Where the matrices of a Muon step lie: ``shapes[i]`` = (rows, cols) of a row-major
    matrix that starts ``offsets[i]`` values into the flat parameter, gradient and average
    buffers, and ``momentum_offsets[i]`` (default: the same) into the momentum buffer.
    Built once per model; holds only the device copy of this table."""

    def __init__(self, shapes, offsets, device, momentum_offsets=None):
        shapes = [(int(r), int(c)) for r, c in shapes]
        offsets = [int(o) for o in offsets]
        moff = list(offsets) if momentum_offsets is None else [int(o) for o in momentum_offsets]
        if not len(shapes) == len(offsets) == len(moff):
            raise ValueError("MuonPlan: one shape, one offset and one momentum offset per matrix expected")
        if any(r < 1 or c < 1 or r >= 1 << 20 or c >= 1 << 20 for r, c in shapes):
            raise ValueError("MuonPlan: 1 to 2^20 - 1 rows and columns expected")
        self.extent = self._extent(shapes, offsets, "offsets")
        self.momentum_extent = self._extent(shapes, moff, "momentum_offsets")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("MuonPlan: a CUDA device expected")
        self.device = torch.device("cuda", torch.cuda.current_device() if device.index is None else device.index)
        by_shape: dict = {}
        for i, s in enumerate(shapes):
            by_shape.setdefault(s, []).append(i)
        # shapes that need a whole GPU first, then the ones of a single CTA in one run, largest first
        single = _lib().muon_single_cta
        rows, self.groups = [], []
        for (r, c), idx in sorted(by_shape.items(), key=lambda kv: (single(*kv[0]), -kv[0][0] * kv[0][1])):
            self.groups += [len(rows), len(idx), r, c]
            rows += [[offsets[i], moff[i], r, c] for i in idx]
        self.count = len(rows)
        self.table = torch.tensor(rows, dtype=torch.int64).reshape(len(rows), 4).to(self.device)

    @staticmethod
    def _extent(shapes, offsets, what) -> int:
        """One past the last value in use; refuses ranges that overlap."""
        end = 0
        for o, (r, c) in sorted(zip(offsets, shapes)):
            if o < 0:
                raise ValueError(f"MuonPlan: negative value in {what}")
            if o < end:
                raise ValueError(f"MuonPlan: two matrices overlap ({what})")
            end = o + r * c
        return end


def muon_step(plan: MuonPlan, data: torch.Tensor, grad: torch.Tensor, momentum_buf: torch.Tensor, *, lr: float,
              wd: float = 0.0, momentum: float = 0.95, nesterov: bool = True, steps: int = 5, eps: float = 1e-7,
              coeffs=NS_COEFFS, adjust_lr: str = "match_rms_adamw", norm_sq: torch.Tensor | None = None,
              max_norm: float = 0.0, skip: torch.Tensor | None = None, ema: torch.Tensor | None = None,
              ema_decay: float = 0.999) -> None:
    """One Muon step in place on the plan's matrices of flat fp32 buffers::

        g = grad * min(1, max_norm / (sqrt(norm_sq) + 1e-6))      (max_norm > 0 and norm_sq given)
        buf = momentum * buf + g;  u = g + momentum * buf  (or buf without nesterov)
        p = p * (1 - lr * wd) - lr * scale(rows, cols) * newton_schulz(u)
        ema = ema + (1 - ema_decay) * (p - ema)                    (ema given)

    ``scale`` is ``0.2 sqrt(max(rows, cols))`` (``"match_rms_adamw"``), ``sqrt(max(1, rows /
    cols))`` (``"original"``) or ``sqrt(max / min)`` (``"nd"``).  ``skip`` (fp32 device value)
    above 0, or a ``norm_sq`` that is not finite, leaves every buffer as it is, decided on the
    device (``norm_sq`` only counts with ``max_norm`` > 0).  Values between the matrices are not
    touched.  The buffers must not overlap one another."""
    if adjust_lr not in _ADJUST:
        raise ValueError(f"unknown adjust_lr {adjust_lr!r}")
    for t, name in ((data, "data"), (grad, "grad"), (momentum_buf, "momentum_buf")):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"muon_step: {name} must be a CUDA tensor")
    if plan.extent > data.numel():
        raise ValueError(f"muon_step: the plan reaches to {plan.extent}, data has {data.numel()} values")
    if plan.momentum_extent > momentum_buf.numel():
        raise ValueError(f"muon_step: the plan reaches to {plan.momentum_extent}, the momentum buffer has "
                         f"{momentum_buf.numel()} values")
    _lib().muon_step(data, grad, momentum_buf, ema, plan.table, plan.groups, float(lr), float(wd), float(momentum),
                     bool(nesterov), int(steps), float(eps), [float(c) for c in coeffs], _ADJUST[adjust_lr], norm_sq,
                     float(max_norm), skip, float(ema_decay), status_word(data.device))
    # written through raw pointers: what autograd saved of them is no longer valid
    torch.autograd.graph.increment_version([data, momentum_buf] if ema is None else [data, momentum_buf, ema])
