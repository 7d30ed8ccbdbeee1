"""Muon over the whole GPU where the work buffers (200 MB of them at a time) make several blocks of
matrices: every matrix gets the bits that it gets alone, some are compared with 64 bits."""

import pytest
import torch
from test_muon_steps_gpu import iterate64, tolerance

pytestmark = pytest.mark.gpu


def test_newton_schulz_in_blocks():
    from synthefy_nori_b200 import ops

    torch.manual_seed(0)
    g = torch.randn(601, 300, 260, device="cuda")  # 0.75 MB a matrix: three blocks
    o = ops.newton_schulz(g)
    for i in range(len(g)):
        assert torch.equal(o[i], ops.newton_schulz(g[i])), i
    for i in (0, 200, 201, 400, 401, 600):
        ref = iterate64(g[i], 5)
        assert float((o[i].double() - ref).norm() / ref.norm()) < tolerance(g[i], 5)


def test_muon_step_in_blocks():
    """Shapes with fewer matrices than there are blocks among one with many."""
    from synthefy_nori_b200 import ops

    torch.manual_seed(1)
    shapes = [(515, 300)] + [(300, 260)] * 601 + [(200, 301)] * 2 + [(64, 64)] * 5
    offsets, n = [], 0
    for r, c in shapes:
        offsets.append(n)
        n += r * c
    p, g, m = (torch.randn(n, device="cuda") * s for s in (0.05, 0.1, 0.3))
    q, v = p.clone(), m.clone()
    ops.muon_step(ops.MuonPlan(shapes, offsets, "cuda"), q, g, v, lr=0.02, wd=0.1)
    for i in [0, 1, 2, 100, 200, 201, 202, 300, 400, 401, 402, 403, 600, 601, 602, 603, 604, 608]:
        (r, c), sl = shapes[i], slice(offsets[i], offsets[i] + shapes[i][0] * shapes[i][1])
        a, b = p[sl].clone(), m[sl].clone()
        ops.muon_step(ops.MuonPlan([(r, c)], [0], "cuda"), a, g[sl].clone(), b, lr=0.02, wd=0.1)
        assert torch.equal(q[sl], a) and torch.equal(v[sl], b), i
        u = (g[sl].double() + 0.95 * (0.95 * m[sl].double() + g[sl].double())).view(r, c)
        upd = 0.02 * 0.2 * max(r, c) ** 0.5 * iterate64(u, 5).flatten()
        tol = tolerance(u, 5) * float(upd.norm()) + 4 * 2.0 ** -24 * float(p[sl].norm() + upd.norm())
        assert float((q[sl].double() - (p[sl].double() * (1 - 0.02 * 0.1) - upd)).norm()) < tol, i
    assert not torch.equal(q, p) and q.isfinite().all() and v.isfinite().all()
