"""Muon operators (orthogonalisation, whole step) against the formulas in 64 bits.

Tolerances.  A step of the iteration rounds five operands to fp16 (the iterate's high part
twice, A twice, C once), each by at most half a step, 2^-11; the polynomial's relative slope
sigma p'(sigma) / p(sigma) is at most 1.2 in modulus on (0, 1.2], so the roundings of five
steps add up without growth: 25 * 2^-11 of the result in the 2-norm.  The result's own
rounding comes on top (half a step of its type).  Weights add three fp32 roundings, the
momentum two products and two sums."""

import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
NS_TOL = 25 * 2.0 ** -11
F32 = 2.0 ** -24


def ns64(g, steps=5, eps=1e-7, coeffs=(A, B, C)):
    a, b, c = coeffs
    x = g.double()
    x = x / (x.flatten(-2).norm(dim=-1)[..., None, None] + eps)
    wide = x.shape[-2] < x.shape[-1]
    x = x.mT if wide else x
    for _ in range(steps):
        s = x.mT @ x
        x = a * x + x @ (b * s + c * (s @ s))
    return x.mT if wide else x


def rel(x, y):
    return float((x.double() - y).norm() / y.norm())


def spectrum(n, m, s, seed=0):
    gen = torch.Generator().manual_seed(seed)
    u = torch.linalg.qr(torch.randn(n, m, generator=gen, dtype=torch.double))[0]
    v = torch.linalg.qr(torch.randn(m, m, generator=gen, dtype=torch.double))[0]
    return ((u * s) @ v).float().cuda()


SHAPES = [(1, 1, 1), (2, 1, 7), (1, 7, 1), (3, 2, 2), (1, 64, 56), (2, 56, 64), (4, 64, 1), (1, 10, 384), (2, 17, 129),
          (1, 128, 128), (2, 384, 128), (1, 129, 128), (3, 255, 33), (1, 448, 64), (1, 999, 96), (2, 333, 127),
          (1, 2000, 17), (1, 130, 1031), (1, 448, 896), (1, 999, 384), (1, 257, 257), (2, 515, 300)]


@pytest.mark.parametrize("batch,rows,cols", SHAPES)
def test_newton_schulz_matches_formula(batch, rows, cols):
    from synthefy_nori_b200 import ops

    torch.manual_seed(rows * 7 + cols)
    g = torch.randn(batch, rows, cols, device="cuda") * torch.logspace(-3, 3, batch, device="cuda")[:, None, None]
    o = ops.newton_schulz(g, out_dtype=torch.float32)
    ref = ns64(g)
    for i in range(batch):
        assert rel(o[i], ref[i]) < NS_TOL
    assert torch.equal(o, ops.newton_schulz(g, out_dtype=torch.float32))  # the same bits again


@pytest.mark.parametrize("rows,cols", [(1, 1), (2, 2), (5, 1), (2, 300), (3, 3), (130, 5), (16, 16), (17, 9), (700, 20),
                                       (32, 32), (31, 400)])
def test_newton_schulz_narrow_matrices_keep_22_bits(rows, cols):
    """Up to 32 columns the products read pairs of fp16: 25 roundings of 2^-22 and as many sums of
    2^-20 at most; the first rounding of the iterate, 2^-22 |G|, is amplified by no more than
    a^5 = 485 in any direction, against a result of norm 0.65 or more."""
    from synthefy_nori_b200 import ops

    torch.manual_seed(rows + 31 * cols)
    g = torch.randn(40, rows, cols, device="cuda")
    o, ref = ops.newton_schulz(g, out_dtype=torch.float32), ns64(g)
    for i in range(40):
        assert rel(o[i], ref[i]) < 25 * (2.0 ** -22 + 2.0 ** -20) + 485 * 2.0 ** -22 / 0.65


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out_dtype", [None, torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(96, 64), (64, 200), (200, 600)])
def test_newton_schulz_types(dtype, out_dtype, rows, cols):
    from synthefy_nori_b200 import ops

    torch.manual_seed(1)
    g = torch.randn(3, rows, cols, device="cuda").to(dtype)
    o = ops.newton_schulz(g, out_dtype=out_dtype)
    assert o.dtype == (out_dtype or dtype) and o.shape == g.shape
    assert rel(o, ns64(g)) < NS_TOL + torch.finfo(o.dtype).eps / 2


@pytest.mark.parametrize("n,m", [(96, 64), (128, 128), (700, 300), (448, 448)])
@pytest.mark.parametrize("kind", ["power1", "power2", "exp", "rank4", "noise"])
def test_newton_schulz_steep_spectra(n, m, kind):
    """Directions far below the largest one keep their place (bf16 iterates would lose them)."""
    from synthefy_nori_b200 import ops

    i = torch.arange(m, dtype=torch.double)
    s = {"power1": 1 / (1 + i), "power2": 1 / (1 + i) ** 2, "exp": 10 ** (-6 * i / m),
         "rank4": (i < 4).double() + 1e-12, "noise": torch.where(i < 8, 1.0, 1e-3)}[kind]
    g = spectrum(n, m, s)
    assert rel(ops.newton_schulz(g), ns64(g)) < NS_TOL


def test_newton_schulz_scale_of_the_gradient():
    """Any fp32 magnitude, a norm far below eps, a zero matrix, and neighbours of a NaN."""
    from synthefy_nori_b200 import ops

    torch.manual_seed(2)
    for rows, cols in ((64, 48), (300, 200)):
        base = torch.randn(rows, cols, device="cuda")
        g = torch.stack([base * k for k in (1e-30, 1e-12, 1e-6, 1.0, 1e30, 0.0, float("nan"), 1.0)])
        g[7, 0, 0] = float("inf")
        o = ops.newton_schulz(g)
        ref = ns64(g[:6])
        for i in range(5):
            assert rel(o[i], ref[i]) < NS_TOL, i
        assert torch.equal(o[5], torch.zeros_like(o[5]))
        assert o[6].isnan().all() and o[7].isnan().all() and o[:6].isfinite().all()


def test_newton_schulz_steps_and_coefficients():
    from synthefy_nori_b200 import ops

    torch.manual_seed(3)
    for shape in ((2, 80, 48), (1, 300, 260)):
        g = torch.randn(*shape, device="cuda")
        for steps in (1, 2, 7):
            assert rel(ops.newton_schulz(g, steps=steps), ns64(g, steps)) < steps * 5 * 2.0 ** -11
        c = (1.875, -1.25, 0.375)  # the convergent quintic
        assert rel(ops.newton_schulz(g, steps=6, coeffs=c), ns64(g, 6, coeffs=c)) < 30 * 2.0 ** -11


def test_newton_schulz_strides_and_batches():
    from synthefy_nori_b200 import ops

    torch.manual_seed(4)
    g = torch.randn(2, 3, 72, 40, device="cuda")
    o = ops.newton_schulz(g)
    assert o.shape == g.shape and rel(o, ns64(g)) < NS_TOL
    t = g.transpose(-1, -2)  # a transposed view: the transposed result
    assert rel(ops.newton_schulz(t), ns64(g).mT) < NS_TOL
    wide = torch.randn(5, 72, 81, device="cuda")[:, :, 3:43]
    assert rel(ops.newton_schulz(wide), ns64(wide)) < NS_TOL
    assert rel(ops.newton_schulz(wide[0]), ns64(wide[0])) < NS_TOL
    assert ops.newton_schulz(g[:0]).shape == (0, 3, 72, 40)
    assert ops.newton_schulz(g[..., :0]).shape == (2, 3, 72, 0)
    h = g.clone()
    assert ops.newton_schulz(h, out=h) is h and torch.equal(h, o)  # in place


def _step64(shapes, offsets, p, g, m, e, *, lr, wd, momentum, nesterov, adjust, clip, decay):
    p, g, m = p.double().clone(), g.double(), m.double().clone()
    e = None if e is None else e.double().clone()
    upd = torch.zeros_like(p)
    for (r, c), o in zip(shapes, offsets):
        sl = slice(o, o + r * c)
        gi = g[sl] * clip
        m[sl] = momentum * m[sl] + gi
        u = gi + momentum * m[sl] if nesterov else m[sl]
        scale = {"match_rms_adamw": 0.2 * max(r, c) ** 0.5, "original": max(1.0, r / c) ** 0.5,
                 "nd": (max(r, c) / min(r, c)) ** 0.5}[adjust]
        upd[sl] = lr * scale * ns64(u.view(r, c)).flatten()
        p[sl] = p[sl] * (1 - lr * wd) - upd[sl]
        if e is not None:
            e[sl] += (1 - decay) * (p[sl] - e[sl])
    return p, m, e, upd


RAGGED = [(64, 64), (192, 64), (64, 1), (1, 1), (10, 96), (2, 96), (333, 127), (448, 64), (64, 64), (300, 200),
          (200, 301), (300, 200), (999, 96), (17, 1500)]  # single-CTA and whole-GPU shapes mixed


def _ragged(seed=0, gap=13, shapes=RAGGED):
    torch.manual_seed(seed)
    off, o = [], 5
    for r, c in shapes:
        off.append(o)
        o += r * c + gap
    n = o + 7
    p, m = torch.randn(n, device="cuda") * 0.05, torch.randn(n, device="cuda") * 0.1
    return shapes, off, p, torch.randn(n, device="cuda") * 0.1, m, p + 0.01


@pytest.mark.parametrize("nesterov,adjust,ema,clip", [(True, "match_rms_adamw", True, True),
                                                      (False, "original", False, False), (True, "nd", False, True)])
def test_muon_step_matches_formula(nesterov, adjust, ema, clip):
    from synthefy_nori_b200 import ops

    shapes, off, p, g, m, e = _ragged()
    e = e if ema else None
    hyper = dict(lr=0.02, wd=0.1, momentum=0.95, nesterov=nesterov)
    norm_sq = g.double().square().sum().float().view(1) if clip else None
    factor = min(1.0, 3.0 / (math.sqrt(float(norm_sq)) + 1e-6)) if clip else 1.0
    ref_p, ref_m, ref_e, upd = _step64(shapes, off, p, g, m, e, **hyper, adjust=adjust, clip=factor, decay=0.9)
    p0, g0 = p.clone(), g.clone()
    plan = ops.MuonPlan(shapes, off, "cuda")
    ops.muon_step(plan, p, g, m, **hyper, adjust_lr=adjust, norm_sq=norm_sq, max_norm=3.0 if clip else 0.0, ema=e,
                  ema_decay=0.9)
    assert torch.equal(g, g0)
    assert ((m - ref_m).abs() <= 4 * F32 * (ref_m.abs() + 2 * g.abs())).all()
    used = torch.zeros_like(p, dtype=torch.bool)
    for (r, c), o in zip(shapes, off):
        sl = slice(o, o + r * c)
        used[sl] = True
        tol = NS_TOL * float(upd[sl].norm()) + 4 * F32 * float(p0[sl].norm() + upd[sl].norm())
        assert float((p[sl].double() - ref_p[sl]).norm()) <= tol, (r, c)
        if ema:
            assert float((e[sl].double() - ref_e[sl]).norm()) <= 0.1 * tol + 4 * F32 * float(ref_e[sl].norm())
    assert torch.equal(p[~used], p0[~used])  # values between the matrices


def test_muon_step_skip_and_bad_norm_leave_everything():
    from synthefy_nori_b200 import ops

    shapes, off, p, g, m, e = _ragged(1)
    plan = ops.MuonPlan(shapes, off, "cuda")
    before = [t.clone() for t in (p, m, e)]
    one, zero = torch.ones(1, device="cuda"), torch.zeros(1, device="cuda")
    for kw in (dict(skip=one), dict(norm_sq=one * float("inf"), max_norm=1.0), dict(norm_sq=one * float("nan"), max_norm=1.0)):
        ops.muon_step(plan, p, g, m, lr=0.1, ema=e, **kw)
        assert all(torch.equal(a, b) for a, b in zip(before, (p, m, e)))
    ops.muon_step(plan, p, g, m, lr=0.1, ema=e, skip=zero)
    assert not torch.equal(before[0], p)


def test_muon_step_momentum_in_its_own_layout():
    from synthefy_nori_b200 import ops

    shapes, off, p, g, m, _ = _ragged(2)
    moff, o = [], 0
    for r, c in shapes:
        moff.append(o)
        o += r * c
    packed = torch.cat([m[o : o + r * c] for (r, c), o in zip(shapes, off)])
    p2, m2 = p.clone(), m.clone()
    ops.muon_step(ops.MuonPlan(shapes, off, "cuda", moff), p, g, packed, lr=0.05)
    ops.muon_step(ops.MuonPlan(shapes, off, "cuda"), p2, g, m2, lr=0.05)
    assert torch.equal(p, p2)
    assert torch.equal(packed, torch.cat([m2[o : o + r * c] for (r, c), o in zip(shapes, off)]))


def test_muon_step_graph_replay_and_two_graphs():
    """Two captured steps of different models replayed in turn: each has its own work buffers."""
    from synthefy_nori_b200 import ops

    runs = []
    for seed in (3, 4):
        shapes, off, p, g, m, e = _ragged(seed)
        plan = ops.MuonPlan(shapes, off, "cuda")
        want = [t.clone() for t in (p, m, e)]
        for _ in range(3):
            ops.muon_step(plan, want[0], g, want[1], lr=0.05, ema=want[2])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            tmp = [t.clone() for t in (p, m, e)]
            ops.muon_step(plan, tmp[0], g, tmp[1], lr=0.05, ema=tmp[2])
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.muon_step(plan, p, g, m, lr=0.05, ema=e)
        runs.append((graph, (p, m, e), want, plan, g))
    for _ in range(3):
        for graph, *_ in runs:
            graph.replay()
    torch.cuda.synchronize()
    for _, got, want, *_ in runs:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_muon_step_with_many_large_shapes():
    """More shapes over the whole GPU than one launch takes, between single-CTA ones."""
    from synthefy_nori_b200 import ops

    shapes = [(130 + 9 * i, 129 + 7 * ((i * 5) % 20)) for i in range(19)] + [(64, 64), (40, 3)]
    shapes = shapes[::2] + shapes[1::2] + [shapes[3]]
    shapes, off, p, g, m, e = _ragged(7, shapes=shapes)
    hyper = dict(lr=0.02, wd=0.1, momentum=0.9, nesterov=True)
    ref_p, _, _, upd = _step64(shapes, off, p, g, m, e, **hyper, adjust="original", clip=1.0, decay=0.9)
    p0 = p.clone()
    ops.muon_step(ops.MuonPlan(shapes, off, "cuda"), p, g, m, **hyper, adjust_lr="original", ema=e, ema_decay=0.9)
    for (r, c), o in zip(shapes, off):
        sl = slice(o, o + r * c)
        tol = NS_TOL * float(upd[sl].norm()) + 4 * F32 * float(p0[sl].norm() + upd[sl].norm())
        assert float((p[sl].double() - ref_p[sl]).norm()) <= tol, (r, c)


def test_empty_plan_and_a_plan_of_one():
    from synthefy_nori_b200 import ops

    flat = torch.ones(8, device="cuda")
    ops.muon_step(ops.MuonPlan([], [], "cuda"), flat, flat.clone(), flat.clone(), lr=0.1)
    assert (flat == 1).all()
    ops.muon_step(ops.MuonPlan([(1, 1)], [7], "cuda"), flat, flat.clone(), flat.clone(), lr=0.1, adjust_lr="original")
    # the iteration on the number 1, five times the quintic
    x = 1.0
    for _ in range(5):
        x = A * x + B * x ** 3 + C * x ** 5
    assert (flat[:7] == 1).all() and abs(float(flat[7]) - (1 - 0.1 * x)) < 1e-5


def test_muon_step_is_ordered_on_its_stream():
    """Large and single-CTA matrices run on two streams inside; the caller's stream sees one call:
    inputs written right before it, results read right after, buffers freed and reused."""
    from synthefy_nori_b200 import ops

    shapes, off, p, g, m, _ = _ragged(8)
    plan = ops.MuonPlan(shapes, off, "cuda")
    want_p, want_m = p.clone(), m.clone()
    for _ in range(6):
        ops.muon_step(plan, want_p, g, want_m, lr=0.02)
        torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        q, n = p.clone(), m.clone()
        for _ in range(6):
            big = torch.full((1 << 24,), 7.0, device="cuda")  # keeps the stream busy, then is freed
            grad = g * 1.0
            ops.muon_step(plan, q, grad, n, lr=0.02)
            grad.fill_(float("nan"))
            del grad, big
            q, n = q.clone(), n.clone()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(q, want_p) and torch.equal(n, want_m)


def test_two_calls_over_the_whole_gpu_at_once():
    from synthefy_nori_b200 import ops

    torch.manual_seed(9)
    gs = [torch.randn(3, 700, 500, device="cuda"), torch.randn(2, 450, 900, device="cuda")]
    want = [ops.newton_schulz(g) for g in gs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(ops.newton_schulz(gs[k]))
    torch.cuda.synchronize()
    ops.check_status(gs[0].device)
    for k in (0, 1):
        assert all(torch.equal(o, want[k]) for o in got[k])


def test_muon_on_a_side_stream_beside_the_default_one():
    from synthefy_nori_b200 import ops

    torch.manual_seed(5)
    a, b = torch.randn(6, 384, 128, device="cuda"), torch.randn(2, 500, 400, device="cuda")
    want_a, want_b = ops.newton_schulz(a), ops.newton_schulz(b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s):
            got_a = ops.newton_schulz(a)
        got_b = ops.newton_schulz(b)
        torch.cuda.synchronize()
        assert torch.equal(got_a, want_a) and torch.equal(got_b, want_b)


def test_hybrid_optimizer_uses_the_kernels():
    """One step of HybridMuonAdamW on the GPU against the same step on the CPU in fp32 with the
    exact orthogonalisation; the checkpoint's form is the same on both."""
    from synthefy_nori_b200.training import muon as tm

    torch.manual_seed(6)
    net = torch.nn.Sequential(torch.nn.Linear(48, 96), torch.nn.GELU(), torch.nn.Linear(96, 130), torch.nn.GELU(),
                              torch.nn.Linear(130, 96))
    ref = copy.deepcopy(net)
    kw = dict(lr=0.01, weight_decay=0.1, ema_decay=0.9, max_grad_norm=0.05)
    ours, theirs = tm.HybridMuonAdamW(net.cuda(), "cuda", **kw), tm.HybridMuonAdamW(ref, "cpu", **kw)
    # the CPU path rounds its iterates to bf16: put the exact iteration there
    plain, tm.newton_schulz = tm.newton_schulz, lambda g, steps=5, eps=1e-7: ns64(g, steps, eps).to(g.dtype)
    try:
        x = torch.randn(64, 48)
        for model, opt, dev in ((net, ours, "cuda"), (ref, theirs, "cpu")):
            opt.zero_grad()
            model(x.to(dev)).pow(2).mean().backward()
            opt.step()
    finally:
        tm.newton_schulz = plain
    for a, b in zip(net.parameters(), ref.parameters()):
        d = float((a.detach().cpu() - b.detach()).norm())
        if b.ndim == 2:  # lr scale |O|, with singular values up to 1.2; gradients differ by fp32 sums
            update = 0.01 * 0.2 * max(b.shape) ** 0.5 * 1.2 * min(b.shape) ** 0.5
            assert d < (NS_TOL + 1e-4) * update + 1e-6 * float(b.detach().norm())
        else:
            assert d < 1e-5
    n = ours.split
    d = float((ours.ema.cpu() - theirs.ema).norm())
    assert d < 0.1 * float((ours.flat.data.cpu() - theirs.flat.data).norm()) + 1e-6 * float(theirs.ema.norm())
    assert n == theirs.split
    sd, sd2 = ours.state_dict(), theirs.state_dict()
    assert [t.shape for t in sd["muon_momentum"]] == [t.shape for t in sd2["muon_momentum"]]
    for a, b in zip(sd["muon_momentum"], sd2["muon_momentum"]):
        assert rel(a.cpu(), b.double()) < 1e-4
    fresh = tm.HybridMuonAdamW(copy.deepcopy(net), "cuda", **kw)
    fresh.load_state_dict(sd)
    for a, b in zip(fresh.state_dict()["muon_momentum"], sd["muon_momentum"]):
        assert torch.equal(a, b)
    before = [p.detach().clone() for p in net.parameters()]
    ours.step(skip=torch.ones((), device="cuda"))
    assert all(torch.equal(a, b) for a, b in zip(before, net.parameters()))


def test_refusals_on_the_gpu():
    from synthefy_nori_b200 import ops

    g = torch.randn(8, 8, device="cuda")
    for bad in (dict(steps=0), dict(steps=65), dict(coeffs=(0.0, 1.0, 1.0)), dict(coeffs=(1.0, 2.0)), dict(eps=-1.0)):
        with pytest.raises(RuntimeError):
            ops.newton_schulz(g, **bad)
    with pytest.raises(ValueError):
        ops.newton_schulz(g, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.newton_schulz(g.double())
    with pytest.raises(ValueError):
        ops.newton_schulz(g[0])
    with pytest.raises(ValueError):
        ops.newton_schulz(g, out=torch.empty(8, 16, device="cuda")[:, ::2])
    plan = ops.MuonPlan([(8, 8)], [3], "cuda")
    flat = torch.zeros(67, device="cuda")
    ops.muon_step(plan, flat, flat.clone(), flat.clone(), lr=0.1)
    with pytest.raises(ValueError):
        ops.muon_step(plan, flat[:66], flat[:66].clone(), flat.clone(), lr=0.1)
    with pytest.raises(ValueError):
        ops.muon_step(plan, flat, flat.clone(), flat[:66].clone(), lr=0.1)
    with pytest.raises(RuntimeError):
        ops.muon_step(plan, flat, flat[:66].clone(), flat.clone(), lr=0.1)
    with pytest.raises(RuntimeError):
        ops.muon_step(plan, flat.double(), flat.clone(), flat.clone(), lr=0.1)
    with pytest.raises(RuntimeError):
        ops.muon_step(plan, flat, flat.clone(), flat.clone(), lr=0.1, skip=torch.zeros((), device="cuda", dtype=torch.int32))
    with pytest.raises(RuntimeError):
        ops.muon_step(plan, flat, flat.clone(), flat.clone(), lr=0.1, ema=flat[:66].clone())
    with pytest.raises(ValueError):
        ops.muon_step(plan, flat, flat.clone(), flat.clone(), lr=0.1, adjust_lr="other")
