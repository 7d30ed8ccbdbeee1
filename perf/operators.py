"""Cases and plain forms of the training operators around the encoder's matrices and rows.

Muon (momentum, orthogonalisation by Newton-Schulz products, weight update) and
LayerNorm (forward, and forward + backward with the weight's gradient).  ``run`` computes
a case with elementary torch operations in 32 bits, or, where ``own`` is true, through
the framework's operators; ``exact`` computes the same from the definitions in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
NS = (3.4445, -4.7750, 2.0315)  # the quintic's coefficients
NS_EPS = 1e-7
LN_EPS = 1e-5
# one optimizer step's settings: the learning rate of the later training tiers, the optimizer's defaults
LR, WD, MOMENTUM, EMA_DECAY, MAX_NORM, STEPS = 1e-4, 0.01, 0.95, 0.999, 1.0, 5

# every matrix that the optimizer gives to Muon, as count x rows x columns, for three presets
TINY = "18x64x64+6x192x64+3x96x64+4x64x32+4x32x64+4x64x1+1x999x96+1x10x96+1x2x96+1x64x48+1x64x2"
NORI_6M = ("51x384x128+32x256x128+49x128x128+17x128x256+34x128x64+64x64x64+32x64x1+1x999x384+1x10x384+1x2x384"
           "+1x64x48+1x128x2")
NORI_100M = ("81x1344x448+52x896x448+79x448x448+27x448x896+53x448x64+52x64x56+52x56x64+52x64x1+1x999x1344+1x10x1344"
             "+1x2x1344+1x128x64+1x64x48+1x448x2")


def listed():
    return [
        # one gate matrix (head width 56): the smallest update there is, where only latency counts
        {"name": "ns_gate", "op": "newton_schulz", "batch": 1, "rows": 64, "cols": 56, "dtype": "float32"},
        # all fused Q/K/V projections of nori-6m
        {"name": "ns_qkv_6m", "op": "newton_schulz", "batch": 51, "rows": 384, "cols": 128, "dtype": "float32"},
        # the quantile head's output matrix: one matrix, odd, wider than tall
        {"name": "ns_head", "op": "newton_schulz", "batch": 1, "rows": 999, "cols": 1344, "dtype": "float32"},
        # all fused Q/K/V projections of nori-100m, from a bf16 gradient
        {"name": "ns_qkv_100m", "op": "newton_schulz", "batch": 81, "rows": 1344, "cols": 448, "dtype": "bfloat16"},
        # the Muon part of one optimizer step: the test preset, the shipped preset, the largest preset
        {"name": "muon_tiny", "op": "muon_step", "shapes": TINY, "nesterov": True, "ema": True},
        {"name": "muon_6m", "op": "muon_step", "shapes": NORI_6M, "nesterov": True, "ema": True},
        {"name": "muon_100m", "op": "muon_step", "shapes": NORI_100M, "nesterov": True, "ema": True},
        # inference on a handful of rows (a label embedding): latency
        {"name": "ln_few", "op": "ln_fwd", "rows": 37, "cols": 64, "dtype": "float32", "out": "float32", "affine": True},
        # a LayerNorm sublayer under bf16 autocast: fp32 results, no affine weight; 16 tables x 1200 rows x 21 tokens
        {"name": "ln_autocast", "op": "ln_fwd", "rows": 403200, "cols": 448, "dtype": "bfloat16", "out": "float32",
         "affine": False},
        # training: the group-fusion norms on every token of a batch, bf16
        {"name": "ln_train_tokens", "op": "ln_train", "rows": 403200, "cols": 448, "dtype": "bfloat16",
         "out": "bfloat16", "affine": True},
        # training in fp32 on an odd number of odd rows
        {"name": "ln_train_odd", "op": "ln_train", "rows": 24001, "cols": 999, "dtype": "float32", "out": "float32",
         "affine": True},
        # training on few wide rows, fp16
        {"name": "ln_train_wide", "op": "ln_train", "rows": 257, "cols": 8192, "dtype": "float16", "out": "float16",
         "affine": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["newton_schulz", "muon_step", "ln_fwd", "ln_train"])
    if op == "newton_schulz":
        rows, cols = _log(rng, 2, 1500), _log(rng, 2, 1500)
        batch = _log(rng, 1, max(1, min(100, 40_000_000 // (rows * cols) // max(1, min(rows, cols) // 448))))
        return {"op": op, "batch": batch, "rows": rows, "cols": cols, "dtype": rng.choice(list(TYPES))}
    if op == "muon_step":
        width, parts, left = _log(rng, 8, 500), [], 30_000_000
        for _ in range(rng.randint(1, 6)):
            r, c = (rng.choice([width, 2 * width, 3 * width, 64, rng.randint(1, 1000)]) for _ in "rc")
            n = max(1, min(_log(rng, 1, 60), left // (r * c)))
            left = max(0, left - n * r * c)
            parts.append(f"{n}x{r}x{c}")
        return {"op": op, "shapes": "+".join(parts), "nesterov": rng.random() < 0.7, "ema": rng.random() < 0.5}
    cols = _log(rng, 8, 9000)
    rows = _log(rng, 1, max(2, min(500_000, 150_000_000 // cols)))
    dtype = rng.choice(list(TYPES))
    return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "out": rng.choice([dtype, "float32"]),
            "affine": rng.random() < 0.7}


def _shapes(case):
    return [tuple(int(v) for v in part.split("x")) for part in case["shapes"].split("+")]


def _gradients(gen, batch, rows, cols):
    """Weight gradients ``dY^T X`` are sums over tokens: a spectrum that falls off, and noise."""
    k = min(rows, cols)
    u = torch.randn(batch, rows, k, device=DEV, generator=gen)
    v = torch.randn(batch, k, cols, device=DEV, generator=gen)
    fall = 1.0 / torch.arange(1, k + 1, device=DEV, dtype=torch.float32)
    size = 10.0 ** (2.0 * torch.rand(batch, 1, 1, device=DEV, generator=gen) - 4.0)
    g = (u * fall) @ v
    return size * (g + 0.05 * torch.randn(batch, rows, cols, device=DEV, generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    if case["op"] == "newton_schulz":
        g = _gradients(gen, case["batch"], case["rows"], case["cols"]).to(TYPES[case["dtype"]])
        return {"case": case, "g": g}
    if case["op"] == "muon_step":
        groups, offsets, shapes, off = [], [], [], 0
        for n, r, c in _shapes(case):
            pitch = -(-r * c // 64) * 64  # every parameter starts on a multiple of 64 values
            groups.append((n, r, c, off, pitch))
            offsets += [off + i * pitch for i in range(n)]
            shapes += [(r, c)] * n
            off += n * pitch
        data, grad, mom = (torch.zeros(off, device=DEV) for _ in range(3))
        for n, r, c, o, pitch in groups:
            at = (n, r, c), (pitch, c, 1), o
            data.as_strided(*at).copy_(torch.randn(n, r, c, device=DEV, generator=gen) * (0.58 / c ** 0.5))
            g = _gradients(gen, n, r, c)
            grad.as_strided(*at).copy_(g)
            mom.as_strided(*at).copy_(4.0 * (g + _gradients(gen, n, r, c)))  # a sum over earlier steps
        ema = data + 1e-3 * data.flip(0) if case["ema"] else None
        state = {"case": case, "groups": groups, "data": data, "grad": grad, "momentum": mom, "ema": ema,
                 "norm_sq": grad.double().square().sum().float().view(1), "skip": torch.zeros(1, device=DEV)}
        if own:
            from synthefy_nori_b200 import ops

            state["plan"] = ops.MuonPlan(shapes, offsets, torch.device(DEV))
        return state
    r, c, t = case["rows"], case["cols"], TYPES[case["dtype"]]
    x = torch.randn(r, c, device=DEV, generator=gen) * (0.5 + torch.rand(r, 1, device=DEV, generator=gen))
    x = (x + torch.randn(r, 1, device=DEV, generator=gen)).to(t)
    w = b = None
    if case["affine"]:
        w = 1.0 + 0.2 * torch.randn(c, device=DEV, generator=gen)
        b = 0.2 * torch.randn(c, device=DEV, generator=gen)
    dy = None
    if case["op"] == "ln_train":
        dy = torch.randn(r, c, device=DEV, generator=gen).to(TYPES[case["out"]])
    return {"case": case, "x": x, "w": w, "b": b, "dy": dy}


def _orthogonalise(g):
    """Five Newton-Schulz products on ``g [batch, rows, cols]`` in 32 bits."""
    a, b, c = NS
    x = g / (g.double().square().sum((1, 2), keepdim=True).sqrt() + NS_EPS).float()
    if x.shape[1] > x.shape[2]:
        x = x.transpose(1, 2)
    for _ in range(STEPS):
        s = x @ x.transpose(1, 2)
        x = a * x + (b * s + c * (s @ s)) @ x
    return x if x.shape[1:] == g.shape[1:] else x.transpose(1, 2)


def _muon_group(s, n, r, c, off, pitch):
    """The plain step on the ``n`` matrices of one shape, in place."""
    at = (n, r, c), (pitch, c, 1), off
    p, g, m = (s[k].as_strided(*at) for k in ("data", "grad", "momentum"))
    clip = (MAX_NORM / (s["norm_sq"].sqrt() + 1e-6)).clamp(max=1.0)
    keep = (s["skip"] <= 0).float()
    g = g * clip
    m.copy_(torch.where(keep > 0, MOMENTUM * m + g, m))
    eff = g + MOMENTUM * m if s["case"]["nesterov"] else m
    new = p * (1.0 - LR * WD) - (LR * 0.2 * max(r, c) ** 0.5) * _orthogonalise(eff)
    p.copy_(torch.where(keep > 0, new, p))
    if s["ema"] is not None:
        e = s["ema"].as_strided(*at)
        e.copy_(torch.where(keep > 0, e + (1.0 - EMA_DECAY) * (p - e), e))


def _ln(s):
    x = s["x"].float()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / ((x - mean).square().mean(1, keepdim=True) + LN_EPS).sqrt()
    h = (x - mean) * rstd
    y = h if s["w"] is None else h * s["w"] + s["b"]
    return y.to(TYPES[s["case"]["out"]]), h, rstd


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["op"] == "newton_schulz":
        return _orthogonalise(state["g"].float()).to(torch.bfloat16)
    if case["op"] == "muon_step":
        for group in state["groups"]:
            _muon_group(state, *group)
        return _muon_out(state)
    y, h, rstd = _ln(state)
    if case["op"] == "ln_fwd":
        return y
    dy = state["dy"].float()
    dh = dy if state["w"] is None else dy * state["w"]
    dx = rstd * (dh - dh.mean(1, keepdim=True) - h * (dh * h).mean(1, keepdim=True))
    out = {"y": y, "dx": dx.to(state["x"].dtype)}
    if state["w"] is not None:
        out["dw"], out["db"] = (dy * h).sum(0), dy.sum(0)
    return out


def _muon_out(state):
    out = {"data": state["data"], "momentum": state["momentum"]}
    if state["ema"] is not None:
        out["ema"] = state["ema"]
    return out


def _run_own(state, case):
    from synthefy_nori_b200 import ops

    if case["op"] == "newton_schulz":
        return ops.newton_schulz(state["g"], steps=STEPS, eps=NS_EPS, coeffs=NS, out_dtype=torch.bfloat16)
    if case["op"] == "muon_step":
        ops.muon_step(state["plan"], state["data"], state["grad"], state["momentum"], lr=LR, wd=WD, momentum=MOMENTUM,
                      nesterov=case["nesterov"], steps=STEPS, eps=NS_EPS, adjust_lr="match_rms_adamw",
                      norm_sq=state["norm_sq"], max_norm=MAX_NORM, skip=state["skip"], ema=state["ema"],
                      ema_decay=EMA_DECAY)
        return _muon_out(state)
    out_t = TYPES[case["out"]]
    y, mean, rstd = ops.layer_norm_fwd(state["x"], state["w"], state["b"], LN_EPS, out_dtype=out_t)
    if case["op"] == "ln_fwd":
        return y
    dx, dw, db = ops.layer_norm_bwd(state["dy"], state["x"], mean, rstd, state["w"], bias_grad=case["affine"])
    out = {"y": y, "dx": dx}
    if case["affine"]:
        out["dw"], out["db"] = dw, db
    return out


def _ns_flops(n, r, c):
    """The three products of each step, the two symmetric ones at half of a full product."""
    m, k = min(r, c), max(r, c)
    return n * STEPS * (m * m * k + m * m * m + 2.0 * m * m * k)


def work(case):
    if case["op"] == "newton_schulz":
        n, r, c = case["batch"], case["rows"], case["cols"]
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": n * r * c * (size + 2), "flops": _ns_flops(n, r, c)}
    if case["op"] == "muon_step":
        values = sum(n * r * c for n, r, c in _shapes(case))
        # gradient in, momentum and weight in and out, the average in and out
        return {"bytes": values * (20 + (8 if case["ema"] else 0)), "flops": sum(_ns_flops(*s) for s in _shapes(case))}
    r, c = case["rows"], case["cols"]
    si, so = (4 if case[k] == "float32" else 2 for k in ("dtype", "out"))
    vec = 8 * c if case["affine"] else 0
    if case["op"] == "ln_fwd":
        return {"bytes": r * c * (si + so) + vec, "flops": 8.0 * r * c}
    # forward: x in, y out; backward: x and dy in, dx out, the two gradients of the weights out
    return {"bytes": r * c * (si + so) + r * c * (2 * si + so) + 2 * vec, "flops": 20.0 * r * c}


def _exact_orthogonal(g):
    """64 bits, on the taller orientation, with the step's polynomial as one matrix."""
    a, b, c = NS
    tall = g.shape[1] >= g.shape[2]
    x = g if tall else g.mT
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + NS_EPS)
    one = torch.eye(x.shape[2], device=x.device, dtype=torch.float64)
    for _ in range(STEPS):
        s = torch.bmm(x.mT, x)
        x = torch.bmm(x, a * one + torch.bmm(s, b * one + c * s))
    return x if tall else x.mT


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "newton_schulz":
        return _exact_orthogonal(s["g"].double())
    if case["op"] == "muon_step":
        out = {k: s[k].double() for k in ("data", "grad", "momentum") + (("ema",) if case["ema"] else ())}
        clip = min(1.0, MAX_NORM / (math.sqrt(float(s["norm_sq"])) + 1e-6))
        for n, r, c, off, pitch in s["groups"]:
            flat = {k: v[off : off + n * pitch].view(n, pitch)[:, : r * c].unflatten(1, (r, c)) for k, v in out.items()}
            g = clip * flat["grad"]
            flat["momentum"].mul_(MOMENTUM).add_(g)
            eff = torch.add(g, flat["momentum"], alpha=MOMENTUM) if case["nesterov"] else flat["momentum"]
            flat["data"].mul_(1.0 - LR * WD).sub_(LR * 0.2 * math.sqrt(max(r, c)) * _exact_orthogonal(eff))
            if case["ema"]:
                flat["ema"].lerp_(flat["data"], 1.0 - EMA_DECAY)
        del out["grad"]
        return out
    x = s["x"].double()
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    inv = (var + LN_EPS).rsqrt()
    w = torch.ones(x.shape[1], device=x.device, dtype=torch.float64) if s["w"] is None else s["w"].double()
    y = (x - mean) * inv * w + (0.0 if s["b"] is None else s["b"].double())
    if case["op"] == "ln_fwd":
        return y
    dy = s["dy"].double()
    xhat = (x - mean) * inv
    # the gradient through the mean and the variance, from dy w alone
    q = dy * w
    proj = torch.einsum("rc,rc->r", q, xhat)[:, None] / x.shape[1]
    out = {"y": y, "dx": inv * (q - q.mean(1, keepdim=True) - proj * xhat)}
    if s["w"] is not None:
        out["dw"], out["db"] = torch.einsum("rc,rc->c", dy, xhat), torch.einsum("rc->c", dy)
    return out
