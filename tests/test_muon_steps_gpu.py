"""Newton-Schulz with any number of steps, in the three forms of the kernels (pairs of fp16, one
CTA a matrix, the whole GPU), against the iteration in 64 bits.

Tolerances.  In the singular basis one step carries an error E of the iterate to E d[i, j], where
d[i, j] are the divided differences of p(s) = a s + b s^3 + c s^5 at (s_i, s_j) for the symmetric
and at (s_i, -s_j) for the skew part, and p(s_j) / s_j for the rows outside; over several steps the
factors multiply.  With u the half step of an operand, a step rounds

    X in A, twice       s (|b| + 2 |c| s^2) 2 u s |X|      (s = max s_i)
    A, twice            s (|b| + 2 |c| s^2) u |A|
    C (or I + C)        a s u |I + C|
    X in the update     a u |X| max|C|

An error spread evenly over the pairs (i, j) grows by the root mean square of their factors.  u is
2^-11 for fp16 operands, whose many roundings are independent of one another: their squares, u^2 / 3
on the average, add over operands and steps.  Up to 32 columns, where operands are pairs, sums fp32
and roundings few, u is 2^-20 and all simply add.  The iterate
keeps 22 bits: 2^-22 of |X_0| = 1 goes through all steps.  Weights and their update are compared
with the same tolerance of the update and fp32's roundings of the weight."""

import pytest
import torch

pytestmark = pytest.mark.gpu

STD = (3.4445, -4.7750, 2.0315)
CONVERGENT = (1.875, -1.25, 0.375)
SHAPES = [(6, 2, 2), (4, 64, 24), (2, 20, 700), (2, 80, 48), (2, 384, 128), (1, 127, 255), (1, 300, 260), (1, 448, 896)]


def iterate64(g, steps, coeffs=STD, eps=1e-7):
    a, b, c = coeffs
    x = g.double()
    x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + eps)
    wide = x.shape[-2] < x.shape[-1]
    x = x.mT if wide else x
    for _ in range(steps):
        s = x.mT @ x
        x = a * x + x @ (b * s + c * (s @ s))
    return x.mT if wide else x


def tolerance(g, steps, coeffs=STD, eps=1e-7):
    """Of one matrix, relative to the result's norm."""
    a, b, c = coeffs
    g = g.double().cpu()
    n, m = max(g.shape), min(g.shape)
    u = 2.0 ** -20 if m <= 32 else 2.0 ** -11
    s = torch.linalg.svdvals(g) / (g.norm() + eps)
    path = [s]
    for _ in range(steps):
        path.append(a * path[-1] + b * path[-1] ** 3 + c * path[-1] ** 5)

    def diff(x, y):  # (p(x) - p(y)) / (x - y)
        return a + b * (x * x + x * y + y * y) + c * (x ** 4 + x ** 3 * y + x * x * y * y + x * y ** 3 + y ** 4)

    sym, skew, out = torch.ones(m, m).double(), torch.ones(m, m).double(), torch.ones(m).double()
    terms = []
    for x in reversed(path[:-1]):
        grow = float(((sym.square().sum() + skew.square().sum()) / 2 + (n - m) * out.square().sum()) / (n * m)) ** 0.5
        A, top, size = x * x, float(x.max()), float(x.norm())
        C = (b * A + c * A * A) / a
        slope = top * (abs(b) + 2 * abs(c) * top ** 2)
        terms += [grow * u * t for t in (slope * 2 * top * size, slope * float(A.norm()), a * top * float((1 + C).norm()),
                                         a * size * float(C.abs().max()))]
        sym, skew = sym * diff(x[:, None], x[None]), skew * diff(x[:, None], -x[None])
        out = out * (a + b * A + c * A * A)
    grow = float(((sym.square().sum() + skew.square().sum()) / 2 + (n - m) * out.square().sum()) / (n * m)) ** 0.5
    start = 2.0 ** -22 * float(s.norm()) * grow
    total = sum(terms) if m <= 32 else (sum(t * t for t in terms) / 3) ** 0.5
    return (total + start) / float(path[-1].norm()) + 2.0 ** -24


def steady(batch, rows, cols, steps, size, eps=1e-7):
    """Matrices of norm ``size`` whose singular values never come near the iteration's repelling fixed
    point 0.868 (there roundings grow until the two sides of it are told apart, in any precision, and
    the factors above say nothing): a relative error of theirs grows by no more than 4 over any number of steps."""
    a, b, c = STD
    gen = torch.Generator().manual_seed(rows * 1009 + cols * 31 + steps)
    n, m = max(rows, cols), min(rows, cols)
    f = size / (size + eps)

    def calm(s):
        x, growth, worst = s * f, torch.ones_like(s), torch.ones_like(s)
        for _ in range(steps):
            y = a * x + b * x ** 3 + c * x ** 5
            d = (x * (a + 3 * b * x * x + 5 * c * x ** 4) / y).abs()
            growth = torch.maximum(d, growth * d)  # the largest product of factors that ends here
            worst, x = torch.maximum(worst, growth), y
        return worst <= 4

    out = []
    for _ in range(1000):
        if len(out) == batch:
            break
        rest = int(torch.randint(1, m // 2 + 1, (1,), generator=gen))  # equal ones that bring the norm to 1
        reach = 0.5 + 0.7 * torch.rand(1, generator=gen, dtype=torch.double)
        s = (0.2 + reach * torch.rand(200 * m, generator=gen, dtype=torch.double)) / m ** 0.5
        s = s[calm(s)][: m - rest]
        last = 1 - s.square().sum()
        if len(s) < m - rest or last <= 0 or not calm((last / rest).sqrt().view(1)):
            continue
        s = torch.cat([s, (last / rest).sqrt().expand(rest)])
        u = torch.linalg.qr(torch.randn(n, m, generator=gen, dtype=torch.double))[0]
        v = torch.linalg.qr(torch.randn(m, m, generator=gen, dtype=torch.double))[0]
        g = size * (u * s) @ v
        out.append(g.mT if rows < cols else g)
    assert len(out) == batch
    return torch.stack(out).float()


def check(o, g, steps, **kw):
    ref = iterate64(g, steps, **kw)
    for i in range(len(g)):
        err = float((o[i].double() - ref[i]).norm() / ref[i].norm())
        assert err < tolerance(g[i], steps, **kw), (i, err)


@pytest.mark.parametrize("batch,rows,cols", SHAPES)
@pytest.mark.parametrize("steps", [1, 6, 10, 12, 16, 20, 40, 64])
def test_many_steps(batch, rows, cols, steps):
    from synthefy_nori_b200 import ops

    g = steady(batch, rows, cols, steps, 3.0).cuda()
    check(ops.newton_schulz(g, steps=steps), g, steps)


@pytest.mark.parametrize("batch,rows,cols", SHAPES)
@pytest.mark.parametrize("steps", [25, 40, 64])
def test_convergent_iteration_to_its_end(batch, rows, cols, steps):
    """The polar factor itself, as far as the steps reach."""
    from synthefy_nori_b200 import ops

    torch.manual_seed(rows + cols + 1)
    g = torch.randn(batch, rows, cols, device="cuda")
    check(ops.newton_schulz(g, steps=steps, coeffs=CONVERGENT), g, steps, coeffs=CONVERGENT)


@pytest.mark.parametrize("rows,cols", [(64, 24), (80, 48), (300, 260)])
@pytest.mark.parametrize("size", [1e-8, 1e-20, 1e-33])
def test_gradients_far_below_eps(rows, cols, size):
    """|G| below eps: the first steps only bring X up to size 1."""
    from synthefy_nori_b200 import ops

    for steps in (5, 24, 64):
        g = steady(1, rows, cols, steps, size).cuda()
        check(ops.newton_schulz(g, steps=steps), g, steps)


@pytest.mark.parametrize("coeffs", [(1.0, 0.0, 0.0), (1.5, -0.5, 0.0), (2.0, -1.5, 0.5)])
def test_other_coefficients(coeffs):
    from synthefy_nori_b200 import ops

    torch.manual_seed(6)
    for shape in ((2, 40, 30), (2, 90, 70), (1, 200, 301)):
        g = torch.randn(*shape, device="cuda")
        for steps in (5, 30, 64):
            check(ops.newton_schulz(g, steps=steps, coeffs=coeffs), g, steps, coeffs=coeffs)


def test_zero_nan_and_infinity_with_many_steps():
    from synthefy_nori_b200 import ops

    torch.manual_seed(7)
    for shape in ((20, 12), (64, 48), (300, 200)):
        g = torch.randn(4, *shape, device="cuda")
        g[1] = 0.0
        g[2, 3, 4] = float("nan")
        g[3, 0, 0] = float("inf")
        o = ops.newton_schulz(g, steps=64)
        assert o[0].isfinite().all() and (o[1] == 0).all() and o[2].isnan().all() and o[3].isnan().all()


@pytest.mark.parametrize("steps", [12, 20, 64])
def test_muon_step_with_many_steps(steps):
    from synthefy_nori_b200 import ops

    shapes = [(64, 24), (80, 48), (384, 128), (300, 260), (200, 301)]
    grads = [steady(1, r, c, steps, 1.0) for r, c in shapes]
    offsets, n = [], 0
    for r, c in shapes:
        offsets.append(n)
        n += r * c
    torch.manual_seed(8)
    p, g = torch.randn(n, device="cuda") * 0.05, torch.cat([x.flatten() for x in grads]).cuda()
    p0, buf, lr, wd = p.double(), torch.zeros(n, device="cuda"), 0.02, 0.1
    ops.muon_step(ops.MuonPlan(shapes, offsets, "cuda"), p, g, buf, lr=lr, wd=wd, steps=steps)
    for (r, c), o in zip(shapes, offsets):
        sl = slice(o, o + r * c)
        u = (g[sl] * 1.95).view(1, r, c)  # the first step's g + momentum g
        upd = lr * 0.2 * max(r, c) ** 0.5 * iterate64(u, steps).flatten()
        tol = tolerance(u[0], steps) * float(upd.norm()) + 4 * 2.0 ** -24 * float(p0[sl].norm() + upd.norm())
        assert float((p[sl].double() - (p0[sl] * (1 - lr * wd) - upd)).norm()) < tol, (r, c)


def test_optimizer_with_many_steps():
    from synthefy_nori_b200.training.muon import HybridMuonAdamW

    torch.manual_seed(9)
    net = torch.nn.Sequential(torch.nn.Linear(48, 96), torch.nn.GELU(), torch.nn.Linear(96, 260)).cuda()
    opt = HybridMuonAdamW(net, "cuda", lr=0.01, ns_steps=20)
    assert opt.plan is not None
    opt.zero_grad()
    net(torch.randn(64, 48, device="cuda")).square().mean().backward()
    opt.step()
    assert all(p.isfinite().all() for p in net.parameters())


def test_refused_coefficients():
    from synthefy_nori_b200 import ops

    g = torch.randn(8, 8, device="cuda")
    for c in ((0.5, 0.0, 0.0), (2000.0, 0.0, 0.0), (-1.0, 0.0, 0.0), (float("nan"), 0.0, 0.0), (2.0, float("inf"), 0.0),
              (2.0, 0.0, float("nan"))):
        with pytest.raises(RuntimeError):
            ops.newton_schulz(g, coeffs=c)
