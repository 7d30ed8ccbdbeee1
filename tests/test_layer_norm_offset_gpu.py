"""LayerNorm on rows of equal values: 2^k of them add up without a rounding, so their mean is the
value itself and the result the bias, as torch's kernel has it."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [2 ** k for k in range(14)])
@pytest.mark.parametrize("pitch", [0, 3])
def test_rows_of_equal_values_give_the_bias(cols, dtype, pitch):
    from synthefy_nori_b200 import ops

    values = torch.tensor([0.1, -1.7, 333.3, 12345.678, 60001.0, 0.0, 1e-4], device="cuda").to(dtype)
    x = torch.empty(7, cols + pitch, device="cuda", dtype=dtype)[:, :cols]  # rows aligned, or not
    x.copy_(values[:, None])
    w, b = torch.randn(cols, device="cuda"), torch.randn(cols, device="cuda")
    y, mean, rstd = ops.layer_norm_fwd(x, w, b, 1e-5, torch.float32)
    assert torch.equal(y, b.expand(7, -1)) and torch.equal(mean, values.float())
    dx, dw, db = ops.layer_norm_bwd(torch.ones_like(y), x, mean, rstd, w, weight_grad=True)
    assert (dw == 0).all() and (db == 7).all() and dx.isfinite().all()
