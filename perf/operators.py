"""Measured cases of the training operators: layer norm, Newton-Schulz orthogonalisation and the Muon step.

Each operator is here in its plain form (elementary torch operations, 32 bits, rounded once at the end) and as the call of the
package's own operator; `exact` has the definitions in 64 bits."""
import math

import torch

own = False

NS = (3.4445, -4.7750, 2.0315)
LN_EPS = 1e-5
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def filters(case):
    """(rows, columns) of the filter matrices of a generator (latent of 128 channels) or a discriminator with `width` base channels."""
    w, k = case["width"], case["layers"]
    if case["model"] == "discriminator":
        chans = [3] + [w * 2 ** i for i in range(k)] + [1]
        return [(o, 16 * i) for i, o in zip(chans, chans[1:])]
    chans = [8 * w, 8 * w, 4 * w, 2 * w, w, w // 2, w // 4][:k + 1]
    blocks = [((o, 9 * i), (o, 9 * o)) + (((o, i),) if i != o else ()) for i, o in zip(chans, chans[1:])]
    return [(8 * w, 9 * 128)] + [s for block in blocks for s in block] + [(3, 9 * chans[-1])]


def listed():
    return [
        # one token's hidden state in a serving loop: latency
        {"name": "ln_token", "op": "ln", "rows": 1, "c": 4096, "dtype": "bf16", "train": False, "act": False, "grid": False},
        # a training batch of tokens of a wide model, forward and backward
        {"name": "ln_train_tokens", "op": "ln", "rows": 16384, "c": 4096, "dtype": "bf16", "train": True, "act": False, "grid": False},
        # the generator's fourth block: 8 images of 3 x 3 patches of 32 x 32 pixels with 52 channels, forward and backward
        {"name": "ln_train_pixels", "op": "ln", "rows": 73728, "c": 52, "dtype": "f32", "train": True, "act": False, "grid": True},
        # its last norm, with the activation behind it: 13 channels in pixels of 16 floats, 128 x 128 pixel patches
        {"name": "ln_pixels_act", "op": "ln", "rows": 1179648, "c": 13, "dtype": "f32", "train": False, "act": True, "grid": True},
        # odd sizes: rows that no vector width divides
        {"name": "ln_train_odd", "op": "ln", "rows": 777, "c": 1021, "dtype": "f16", "train": True, "act": False, "grid": False},
        # the per-head matrices of an attention layer
        {"name": "ns_heads", "op": "ns", "batch": 16, "m": 64, "n": 64, "dtype": "bf16"},
        # the widest filter of the discriminator
        {"name": "ns_filter", "op": "ns", "batch": 1, "m": 512, "n": 4096, "dtype": "f32"},
        # odd sizes, more rows than columns
        {"name": "ns_tall_odd", "op": "ns", "batch": 2, "m": 1501, "n": 333, "dtype": "bf16"},
        # a large projection in 32 bits and one in bfloat16
        {"name": "ns_large", "op": "ns", "batch": 1, "m": 4096, "n": 4096, "dtype": "f32"},
        {"name": "ns_large_wide", "op": "ns", "batch": 1, "m": 4096, "n": 8192, "dtype": "bf16"},
        # an optimiser step on all filters of the default generator, and of the default discriminator
        {"name": "muon_generator", "op": "muon", "model": "generator", "width": 52, "layers": 6, "ema": True},
        {"name": "muon_discriminator", "op": "muon", "model": "discriminator", "width": 64, "layers": 4, "ema": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("ln", "ln", "ns", "ns", "muon"))
    if op == "ln":
        dtype = rng.choice(("f32", "bf16", "f16"))
        grid = dtype == "f32" and rng.random() < 0.4
        c = _log(rng, 3, 512) if grid else _log(rng, 16, 40000)
        rows = _log(rng, 1, max(1, (60 << 20) // c))
        train = rng.random() < 0.6
        return {"op": "ln", "rows": min(rows, 1200000), "c": c, "dtype": dtype, "train": train, "act": not train and rng.random() < 0.5,
                "grid": grid}
    if op == "ns":
        m, n = _log(rng, 8, 4096), _log(rng, 8, 8192)
        if rng.random() < 0.3:
            m, n = n, m
        most = 5e10 / (min(m, n) ** 2 * max(m, n))
        return {"op": "ns", "batch": min(24, max(1, _log(rng, 1, max(1.0, most)))), "m": m, "n": n, "dtype": rng.choice(("f32", "bf16", "f16"))}
    if rng.random() < 0.5:
        return {"op": "muon", "model": "generator", "width": rng.randint(8, 52), "layers": rng.randint(4, 6), "ema": rng.random() < 0.5}
    return {"op": "muon", "model": "discriminator", "width": rng.randint(8, 64), "layers": rng.randint(3, 5), "ema": rng.random() < 0.5}


def _rand(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _gradient(gen, *shape):
    """What a layer's gradient looks like: a few strong directions over a broad floor."""
    k = min(16, *shape[-2:])
    return 1e-3 * (_rand(gen, *shape) + _rand(gen, *shape[:-1], k) @ _rand(gen, *shape[:-2], k, shape[-1]).contiguous())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "ln":
        rows, c, t = case["rows"], case["c"], DTYPES[case["dtype"]]
        ld = (c + 3) // 4 * 4 if case["grid"] else c
        x = _rand(gen, rows, c) * (0.5 + _rand(gen, c).abs()) + _rand(gen, c)
        x = torch.nn.functional.pad(x, (0, ld - c)).to(t)
        dy = torch.nn.functional.pad(_rand(gen, rows, c) * 0.1, (0, ld - c)).to(t) if case["train"] else None
        if case["grid"]:      # patch-grid pixels: (images, grid rows, grid columns, patch rows, patch columns, floats per pixel)
            x = x.view(rows, 1, 1, 1, 1, ld)
            dy = dy.view(rows, 1, 1, 1, 1, ld) if case["train"] else None
        w, b = (1 + 0.2 * _rand(gen, c)).to(t), (0.2 * _rand(gen, c)).to(t)
        if case["train"]:
            x, w, b = x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
        return {"case": case, "x": x, "w": w, "b": b, "dy": dy}
    if case["op"] == "ns":
        g = _gradient(gen, case["batch"], case["m"], case["n"])
        return {"case": case, "g": g.to(DTYPES[case["dtype"]])}
    shapes = filters(case)
    g = torch.cat([_gradient(gen, m, n).reshape(-1) for m, n in shapes])
    mom = torch.cat([_gradient(gen, m, n).reshape(-1) for m, n in shapes])
    p = 0.05 * _rand(gen, g.numel())
    ema = p + 1e-3 * _rand(gen, g.numel()) if case["ema"] else None
    state = {"case": case, "p": p, "g": g, "m": mom, "ema": ema}
    if own:
        from infinite_texture_gans_amd import ops
        state["plan"] = ops.MuonPlan(shapes, g.device)
    return state


SLOPE = 0.2
MUON = {"lr": 0.02, "momentum": 0.95, "weight_decay": 0.01, "ema_decay": 0.999}


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    with torch.no_grad():
        if case["op"] == "ln":
            return _plain_ln(case, state["x"], state["w"], state["b"], state["dy"])
        if case["op"] == "ns":
            return _plain_ns(state["g"].float()).to(state["g"].dtype)
        return _plain_muon(case, state)


def _run_own(case, s):
    from infinite_texture_gans_amd import ops
    if case["op"] == "ln":
        x = ops.GT(s["x"], case["c"]) if case["grid"] else s["x"]
        y = ops.layer_norm(x, s["w"], s["b"], eps=LN_EPS, act=ops.ACT_LRELU if case["act"] else ops.ACT_NONE, slope=SLOPE)
        y = y.t if case["grid"] else y
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
    if case["op"] == "ns":
        return ops.orthogonalize(s["g"])
    ops.muon_step(s["plan"], s["p"], s["g"], s["m"], s["ema"], nesterov=True, **MUON)
    return [t for t in (s["p"], s["m"], s["ema"]) if t is not None]


def _plain_ln(case, x, w, b, dy):
    c, t, shape = case["c"], x.dtype, x.shape
    z = x.reshape(-1, shape[-1])[:, :c].float()
    wf, bf = w.float(), b.float()
    d = z - z.mean(1, keepdim=True)
    r = torch.rsqrt((d * d).mean(1, keepdim=True) + LN_EPS)
    xh = d * r
    y = xh * wf + bf
    if case["act"]:
        y = torch.where(y > 0, y, SLOPE * y)
    pad = (0, shape[-1] - c)
    y = torch.nn.functional.pad(y, pad).to(t).view(shape)
    if not case["train"]:
        return y
    du = dy.reshape(-1, shape[-1])[:, :c].float()
    g = du * wf
    dx = r * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return y, torch.nn.functional.pad(dx, pad).to(t).view(shape), (du * xh).sum(0).to(w.dtype), du.sum(0).to(b.dtype)


def _plain_ns(g):
    """Matrices (..., m, n) in 32 bits; the norm is a long sum and is taken in 64."""
    norm = g.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = (g / norm).float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    a, b, c = NS
    for _ in range(5):
        s = x @ x.mT.contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.mT.contiguous() if tall else x


def _plain_muon(case, s):
    mu, lr = MUON["momentum"], MUON["lr"]
    s["m"].mul_(mu).add_(s["g"])
    u = s["g"] + mu * s["m"]
    at = 0
    upd = torch.empty_like(u)
    for m, n in filters(case):
        upd[at:at + m * n] = math.sqrt(max(1.0, m / n)) * _plain_ns(u[at:at + m * n].view(m, n)).reshape(-1)
        at += m * n
    s["p"].mul_(1 - lr * MUON["weight_decay"]).sub_(lr * upd)
    if s["ema"] is not None:
        s["ema"].mul_(MUON["ema_decay"]).add_((1 - MUON["ema_decay"]) * s["p"])
    return [t for t in (s["p"], s["m"], s["ema"]) if t is not None]


def work(case):
    if case["op"] == "ln":
        n, e = case["rows"] * case["c"], 4 if case["dtype"] == "f32" else 2
        # forward: x in, y out; backward: x and dy in, dx out; the gain and the shift, and their gradients
        return {"bytes": (5 if case["train"] else 2) * n * e + (4 if case["train"] else 2) * case["c"] * e, "flops": (22 if case["train"] else 8) * n}

    def ns(m, n):
        m, n = min(m, n), max(m, n)
        return 5.0 * (3 * m * m * n + m * m * m)
    if case["op"] == "ns":
        e = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * e * case["batch"] * case["m"] * case["n"], "flops": case["batch"] * ns(case["m"], case["n"])}
    shapes = filters(case)
    return {"bytes": (7 if case["ema"] else 5) * 4 * sum(m * n for m, n in shapes), "flops": sum(ns(m, n) for m, n in shapes)}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ln":
            return _exact_ln(case, s)
        if case["op"] == "ns":
            return torch.stack([_exact_polar(g.double()) for g in s["g"]])
        g, mom, p = s["g"].double(), s["m"].double(), s["p"].double()
        mom = MUON["momentum"] * mom + g
        parts, shapes = [], filters(case)
        for (m, n), u in zip(shapes, torch.split(g + MUON["momentum"] * mom, [m * n for m, n in shapes])):
            parts.append((_exact_polar(u.view(m, n)) * max(1.0, m / n) ** 0.5).flatten())
        p = p - MUON["lr"] * (MUON["weight_decay"] * p + torch.cat(parts))
        d = MUON["ema_decay"]
        return [p, mom] + ([d * s["ema"].double() + (1 - d) * p] if case["ema"] else [])


def _exact_ln(case, s):
    c, shape = case["c"], s["x"].shape
    z, w, b = s["x"].detach().flatten(0, -2)[:, :c].double(), s["w"].detach().double(), s["b"].detach().double()
    std = torch.sqrt(z.var(1, unbiased=False, keepdim=True) + LN_EPS)
    xh = (z - z.mean(1, keepdim=True)) / std

    def whole(v):
        out = torch.zeros(v.shape[0], shape[-1], device=v.device, dtype=v.dtype)
        out[:, :c] = v
        return out.view(shape)
    y = w * xh + b
    if case["act"]:
        y = torch.maximum(y, SLOPE * y)
    if not case["train"]:
        return whole(y)
    dy = s["dy"].flatten(0, -2)[:, :c].double()
    q = w * dy
    dx = (c * q - q.sum(1, keepdim=True) - xh * (q * xh).sum(1, keepdim=True)) / (c * std)
    return whole(y), whole(dx), torch.einsum("rc,rc->c", dy, xh), dy.sum(0)


def _exact_polar(g):
    """Five odd-polynomial steps on the singular values, as products of the matrix itself."""
    x = g / torch.linalg.matrix_norm(g)
    a, b, c = NS
    for _ in range(5):
        gram = x @ x.T if g.shape[0] <= g.shape[1] else x.T @ x
        eye = torch.eye(gram.shape[0], device=g.device, dtype=g.dtype)
        poly = a * eye + gram @ (b * eye + c * gram)
        x = poly @ x if g.shape[0] <= g.shape[1] else x @ poly
    return x
