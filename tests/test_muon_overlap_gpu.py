"""Buffers of the Muon operators that share memory: in place as documented, refused otherwise."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols", [(20, 12), (200, 300)])
def test_newton_schulz_in_place_or_apart(rows, cols):
    from synthefy_nori_b200 import ops

    torch.manual_seed(0)
    n = rows * cols
    flat = torch.randn(5 * n, device="cuda")
    g = flat[: 3 * n].view(3, rows, cols)
    want = ops.newton_schulz(g)
    for start in (1, 4, n, 3 * n - 1):  # from one value to all but one off
        with pytest.raises(RuntimeError, match="share no memory"):
            ops.newton_schulz(g, out=flat[start : start + 3 * n].view_as(g) if start + 3 * n <= 5 * n else flat[-3 * n :].view_as(g))
    low = flat.view(torch.bfloat16)[: 3 * n].view(3, rows, cols)  # g's first half, seen as another type
    with pytest.raises(RuntimeError, match="share no memory"):
        ops.newton_schulz(g, out=low)
    with pytest.raises(RuntimeError, match="share no memory"):
        ops.newton_schulz(low, out=g)
    behind = torch.empty(6 * n, device="cuda")  # neighbours in one allocation
    behind[: 3 * n].copy_(g.flatten())
    out = behind[3 * n :].view_as(g)
    assert torch.equal(ops.newton_schulz(behind[: 3 * n].view_as(g), out=out), want)
    assert torch.equal(behind[: 3 * n].view_as(g), g)
    assert ops.newton_schulz(g, out=g) is g and torch.equal(g, want)


def test_muon_step_buffers_apart():
    from synthefy_nori_b200 import ops

    torch.manual_seed(1)
    plan = ops.MuonPlan([(8, 8)], [0], "cuda")
    big = torch.randn(256, device="cuda")
    a, b, c, d = big.split(64)  # neighbours: fine
    e = big[32:96]
    for bad in ((a, a, b, None), (a, b, a, None), (a, b, b, None), (a, b, c, a), (a, b, c, b), (a, b, c, c), (a, e, c, None),
                (a, c, e, None), (a, c, d, e)):
        before = big.clone()
        with pytest.raises(RuntimeError, match="share memory"):
            ops.muon_step(plan, *bad[:3], lr=0.1, ema=bad[3])
        assert torch.equal(big, before)
    want = [t.clone() for t in (a, b, c, d)]
    ops.muon_step(plan, want[0], want[1], want[2], lr=0.1, ema=want[3])
    ops.muon_step(plan, a, b, c, lr=0.1, ema=d)
    assert all(torch.equal(x, y) for x, y in zip((a, b, c, d), want))
