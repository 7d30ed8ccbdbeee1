"""The model's LayerNorm modules and the operators on CUDA tensors that have no memory (fake tensors
need no GPU): the modules take torch's path, the operators refuse."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from synthefy_nori_b200 import ops
from synthefy_nori_b200.models.layers import LayerNorm, LayerNormMixedPrecision


def test_is_plain():
    x = torch.zeros(3)
    assert ops.is_plain(x) and ops.is_plain(torch.nn.Parameter(x))
    seen = []
    torch.func.vmap(lambda t: (seen.append(ops.is_plain(t)), t)[1])(torch.zeros(2, 3))
    torch.func.grad(lambda t: (seen.append(ops.is_plain(x)), t.sum())[1])(x)
    with torch.autograd.forward_ad.dual_level():
        seen.append(ops.is_plain(x))
    with FakeTensorMode() as mode:
        seen.append(ops.is_plain(x))
        fake = torch.zeros(3, device="cuda")
    seen.append(ops.is_plain(fake))
    torch.jit.trace(lambda t: (seen.append(ops.is_plain(t)), t + 1)[1], x, check_trace=False)
    assert mode is not None and seen == [False] * 6 and ops.is_plain(x)


@pytest.mark.parametrize("cls", [LayerNorm, LayerNormMixedPrecision])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_modules_on_fake_cuda_tensors(cls, dtype):
    with FakeTensorMode():
        m = cls(24, device="cuda", dtype=dtype)
        x = torch.empty(5, 24, device="cuda", dtype=dtype)
        y = m(x)
        assert y.shape == x.shape and y.dtype == dtype and y.device == x.device
    assert m(x).shape == x.shape  # outside of the mode, too


def test_operators_refuse_fake_tensors():
    with FakeTensorMode():
        x, w = torch.empty(6, 8, device="cuda"), torch.empty(8, device="cuda")
        flat, row = torch.empty(48, device="cuda"), torch.empty(6, device="cuda")
    lib = ops.lib()
    with pytest.raises(RuntimeError, match="plain tensor"):
        ops.layer_norm(x, w, w)
    with pytest.raises(RuntimeError, match="plain tensor"):
        ops.layer_norm_fwd(x, w, w)
    with pytest.raises(RuntimeError, match="plain tensor"):
        ops.layer_norm_bwd(x, x, row, row, w)
    with pytest.raises(RuntimeError, match="plain tensor"):
        lib.newton_schulz(x, None, None, 5, 1e-7, ops.NS_COEFFS, flat)
    with pytest.raises(RuntimeError, match="plain tensor"):
        lib.muon_step(flat, flat, flat, None, flat, [0, 1, 6, 8], 0.1, 0.0, 0.9, True, 5, 1e-7, list(ops.NS_COEFFS), 0,
                      None, 0.0, None, 0.9, flat)


@pytest.mark.parametrize("wrap", [torch.func.vmap, lambda f: torch.func.grad(lambda x: f(x).sum())])
def test_cpu_modules_under_transforms(wrap):
    x = torch.randn(4, 5, 24)
    m, t = LayerNorm(24), torch.nn.LayerNorm(24)
    assert torch.equal(wrap(m)(x), wrap(t)(x))
