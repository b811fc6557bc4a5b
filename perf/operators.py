"""
Workloads of the half-precision dense layer and of the matrix optimizer, each
with its plain form in elementary torch operations.

- ``linear``: y = f(x W^T + b) + r in bf16 or fp16 (f one of none, relu, silu,
  gelu), forward alone or with its backward (dx, dW, db, dr).
- ``newton_schulz``: the orthogonalised update of a stack of matrices.
- ``muon``: one optimizer step over a flat buffer of matrices (momentum,
  Newton-Schulz products, weight decay, update), in place.

Sizes are those of the 85M model and the small MLIP of create_graph_b200.mlip
(8280 atoms of the headline workload; 768 and 128 channels; 3072 and 512 in the
feed-forward layer), and generic ones: one row, odd sizes, long batches.
"""

import math

import torch

own = False

HALF = {"bf16": torch.bfloat16, "fp16": torch.float16}
DTYPES = {**HALF, "fp32": torch.float32}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
LR, MOMENTUM, WEIGHT_DECAY = 1e-3, 0.95, 0.1
# a flat buffer's slices start on 256-byte boundaries: 64 fp32 values
ALIGN = 64
LARGEST_LINEAR = 65536 * 768 * 3072


def listed():
    return [
        # one atom through the first feed-forward layer: a single row, latency
        {"name": "linear 1 row", "op": "linear", "m": 1, "k": 768, "n": 3072, "dtype": "bf16", "act": "silu",
         "bias": True, "residual": False, "train": False},
        # a small system through the small MLIP's second layer, with gradients: launches count
        {"name": "linear 64 rows train", "op": "linear", "m": 64, "k": 512, "n": 128, "dtype": "fp16", "act": "none",
         "bias": True, "residual": True, "train": True},
        # the headline workload's second feed-forward layer into the residual stream
        {"name": "linear ffn2 residual", "op": "linear", "m": 8280, "k": 3072, "n": 768, "dtype": "bf16",
         "act": "none", "bias": True, "residual": True, "train": False},
        # the headline workload's first feed-forward layer, with gradients
        {"name": "linear ffn1 silu train", "op": "linear", "m": 8280, "k": 768, "n": 3072, "dtype": "bf16",
         "act": "silu", "bias": True, "residual": False, "train": True},
        # odd sizes: rows, inner and outer lengths that no tile or 16-byte row divides
        {"name": "linear odd gelu train", "op": "linear", "m": 4099, "k": 515, "n": 1031, "dtype": "fp16",
         "act": "gelu", "bias": True, "residual": True, "train": True},
        # a long batch of atoms through the same layer
        {"name": "linear 65536 rows train", "op": "linear", "m": 65536, "k": 768, "n": 3072, "dtype": "bf16",
         "act": "gelu", "bias": True, "residual": True, "train": True},
        # the small MLIP's square matrices: a chain of tiny products
        {"name": "newton_schulz 4x128x128", "op": "newton_schulz", "batch": 4, "rows": 128, "cols": 128,
         "dtype": "fp32"},
        # one tall matrix of the 85M model in half precision
        {"name": "newton_schulz 3072x768", "op": "newton_schulz", "batch": 1, "rows": 3072, "cols": 768,
         "dtype": "bf16"},
        # odd sizes
        {"name": "newton_schulz odd", "op": "newton_schulz", "batch": 3, "rows": 257, "cols": 1031, "dtype": "fp32"},
        # every output projection of the 85M model
        {"name": "newton_schulz 12x768x768", "op": "newton_schulz", "batch": 12, "rows": 768, "cols": 768,
         "dtype": "fp32"},
        # the small MLIP's matrices (4 blocks) in one step
        {"name": "muon small", "op": "muon", "blocks": 4, "hidden": 128, "ffn": 512},
        # the 85M model's matrices (12 blocks) in one step
        {"name": "muon 85m", "op": "muon", "blocks": 12, "hidden": 768, "ffn": 3072},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "newton_schulz", "newton_schulz", "muon"])
    if op == "linear":
        k, n = _log(rng, 16, 4096), _log(rng, 16, 4096)
        if rng.random() < 0.5:
            k, n = -(-k // 8) * 8, -(-n // 8) * 8
        return {"op": op, "m": _log(rng, 1, min(65536, LARGEST_LINEAR // (k * n))), "k": k, "n": n,
                "dtype": rng.choice(["bf16", "fp16"]), "act": rng.choice(["none", "relu", "silu", "gelu"]),
                "bias": rng.random() < 0.7, "residual": rng.random() < 0.5, "train": rng.random() < 0.5}
    if op == "newton_schulz":
        rows, cols = _log(rng, 16, 3000), _log(rng, 16, 3000)
        case = {"op": op, "batch": 1, "rows": rows, "cols": cols, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
        most = int(work(listed()[-1])["flops"] / work(case)["flops"])
        case["batch"] = _log(rng, 1, max(1, min(16, most)))
        return case
    hidden = _log(rng, 48, 768)
    return {"op": op, "blocks": rng.randint(1, 12), "hidden": hidden, "ffn": _log(rng, hidden, 4 * hidden)}


def _shapes(case):
    """The matrices of the model's blocks: q/k/v, output projection, feed-forward."""
    c, f = case["hidden"], case["ffn"]
    return [(3 * c, c), (c, c), (f, c), (c, f)] * case["blocks"]


def _offsets(shapes):
    """(start of each matrix, length) of a flat buffer with aligned slices."""
    starts, at = [], 0
    for r, c in shapes:
        starts.append(at)
        at += -(-(r * c) // ALIGN) * ALIGN
    return starts, at


def _views(flat, shapes):
    return [flat[s : s + r * c].view(r, c) for s, (r, c) in zip(_offsets(shapes)[0], shapes)]


def _gradient(shape, scale, gen):
    """What the gradient of a dense layer looks like: a few strong directions
    (a sum over correlated rows) over noise."""
    *batch, r, c = shape
    k = max(1, min(32, r // 2, c // 2))
    strong = torch.randn(*batch, r, k, generator=gen, device="cuda") @ torch.randn(*batch, k, c, generator=gen,
                                                                                   device="cuda")
    return scale * (strong / math.sqrt(k) + torch.randn(*batch, r, c, generator=gen, device="cuda"))


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (scale * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)

    if case["op"] == "linear":
        m, k, n, dt = case["m"], case["k"], case["n"], HALF[case["dtype"]]
        s = {"x": normal(m, k, dtype=dt), "weight": normal(n, k, scale=1.0 / math.sqrt(k), dtype=dt),
             "bias": normal(n, scale=0.5, dtype=dt) if case["bias"] else None,
             "residual": normal(m, n, dtype=dt) if case["residual"] else None}
        if case["train"]:
            s["grad"] = normal(m, n, scale=0.1, dtype=dt)
        return s
    if case["op"] == "newton_schulz":
        return {"x": _gradient((case["batch"], case["rows"], case["cols"]), 1e-3, gen).to(DTYPES[case["dtype"]])}
    shapes = _shapes(case)
    total = _offsets(shapes)[1]
    s = {name: torch.zeros(total, device="cuda") for name in ("weight", "grad", "momentum")}
    for w, g, b in zip(*(_views(s[name], shapes) for name in ("weight", "grad", "momentum"))):
        w.copy_(normal(*w.shape, scale=1.0 / math.sqrt(w.shape[1])))
        g.copy_(_gradient(g.shape, 1e-3, gen))
        b.copy_(_gradient(b.shape, 1e-3, gen))
    return s


def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    if case["op"] == "linear" and case["train"]:
        for name in ("x", "weight", "bias", "residual"):
            if state[name] is not None:
                state[name].requires_grad_(True)
    if case["op"] == "muon" and own:
        # the optimizer that a training program keeps, on the same values
        from create_graph_b200.ddp import FlatGradients
        from create_graph_b200.optim import FusedMuon

        shapes = _shapes(case)
        params = [torch.nn.Parameter(w) for w in _views(state["weight"], shapes)]
        grads = FlatGradients(params, None)
        grads.flat.copy_(state["grad"])
        opt = FusedMuon(grads, lr=LR, momentum=MOMENTUM, weight_decay=WEIGHT_DECAY, steps=STEPS,
                        coefficients=COEFFICIENTS, eps=EPS)
        opt.momentum_buffer.copy_(state["momentum"])
        state = {"case": dict(case), "optimizer": opt}
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------


def _act(z, name):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp_min(0.0)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _act_grad(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)


def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    x, w = s["x"].detach().float(), s["weight"].detach().float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].detach().float()
    y = _act(z, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].detach().float()
    out = {"y": y.to(dt)}
    if case["train"]:
        g = s["grad"].float()
        gz = g if case["act"] == "none" else g * _act_grad(z, case["act"])
        out["dx"], out["dw"] = (gz @ w).to(dt), (gz.t() @ x).to(dt)
        if s["bias"] is not None:
            out["db"] = gz.sum(0).to(dt)
        if s["residual"] is not None:
            out["dr"] = s["grad"]
    return out


def _plain_newton_schulz(x):
    a, b, c = COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if tall else x


def _plain_muon(s):
    """m <- m + (1 - mu) (g - m); u = g + mu (m - g); W <- (1 - lr wd) W - lr scale NS(u)."""
    shapes = _shapes(s["case"])
    m = s["momentum"].lerp_(s["grad"], 1.0 - MOMENTUM)
    update = _views(s["grad"].lerp(m, MOMENTUM), shapes)
    weights = _views(s["weight"].mul_(1.0 - LR * WEIGHT_DECAY), shapes)
    for shape in dict.fromkeys(shapes):  # equal shapes in one stack
        at = [i for i, other in enumerate(shapes) if other == shape]
        rate = LR * math.sqrt(max(1.0, shape[0] / shape[1]))
        steps = _plain_newton_schulz(torch.stack([update[i] for i in at]))
        torch._foreach_add_([weights[i] for i in at], list(steps), alpha=-rate)
    return {"weight": s["weight"], "momentum": m}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _own_linear(s):
    from create_graph_b200.dense import linear

    y = linear(s["x"], s["weight"], s["bias"], activation=s["case"]["act"], residual=s["residual"])
    if not s["case"]["train"]:
        return {"y": y}
    leaves = {"dx": s["x"], "dw": s["weight"], "db": s["bias"], "dr": s["residual"]}
    leaves = {name: leaf for name, leaf in leaves.items() if leaf is not None}
    grads = torch.autograd.grad(y, list(leaves.values()), s["grad"])
    return {"y": y, **dict(zip(leaves, grads))}


def run(state):
    op = state["case"]["op"]
    if not own:
        if op == "linear":
            return _plain_linear(state)
        if op == "newton_schulz":
            return _plain_newton_schulz(state["x"].float()).to(state["x"].dtype)
        return _plain_muon(state)
    if op == "linear":
        return _own_linear(state)
    if op == "newton_schulz":
        from create_graph_b200.optim import newton_schulz

        return newton_schulz(state["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    opt = state["optimizer"]
    opt.step()
    return {"weight": opt.flat, "momentum": opt.momentum_buffer}


def _newton_schulz_flops(rows, cols):
    """Per step the two symmetric products' lower halves (s^2 l and s^3) and B X (2 s^2 l)."""
    s, l = min(rows, cols), max(rows, cols)
    return STEPS * (3.0 * s * s * l + 1.0 * s * s * s)


def work(case):
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        values = m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        flops = 2.0 * m * k * n
        if case["train"]:
            # the gradient in, dx, dW and db out (dr is the gradient itself)
            values += m * n + m * k + n * k + (n if case["bias"] else 0)
            flops *= 3.0
        return {"bytes": 2.0 * values, "flops": flops}
    if case["op"] == "newton_schulz":
        values = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2.0 * (4 if case["dtype"] == "fp32" else 2) * values,
                "flops": case["batch"] * _newton_schulz_flops(case["rows"], case["cols"])}
    shapes = _shapes(case)
    # gradient in, momentum and weight in and out
    return {"bytes": 20.0 * sum(r * c for r, c in shapes), "flops": sum(_newton_schulz_flops(r, c) for r, c in shapes)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _orthogonalised(g):
    """The update of one matrix in 64 bits, through its own sides: on the left
    of a wide matrix, on the right of a tall one."""
    a, b, c = COEFFICIENTS
    g = g.double()
    x = g / max(float(torch.linalg.vector_norm(g)), EPS)
    wide = x.shape[0] <= x.shape[1]
    for _ in range(STEPS):
        if wide:
            p = torch.mm(x, x.t())
            x = a * x + torch.mm(b * p + c * torch.mm(p, p), x)
        else:
            p = torch.mm(x.t(), x)
            x = a * x + torch.mm(x, b * p + c * torch.mm(p, p))
    return x


def exact(case, seed):
    s = {name: v.double() if v is not None else None for name, v in _inputs(case, seed).items()}
    if case["op"] == "newton_schulz":
        return torch.stack([_orthogonalised(m) for m in s["x"]])
    if case["op"] == "muon":
        shapes = _shapes(case)
        m = MOMENTUM * s["momentum"] + (1.0 - MOMENTUM) * s["grad"]
        u = (1.0 - MOMENTUM) * s["grad"] + MOMENTUM * m
        w = (1.0 - LR * WEIGHT_DECAY) * s["weight"]
        for (rows, cols), to, frm in zip(shapes, _views(w, shapes), _views(u, shapes)):
            to -= LR * max(1.0, rows / cols) ** 0.5 * _orthogonalised(frm)
        return {"weight": w, "momentum": m}
    z = torch.nn.functional.linear(s["x"], s["weight"], s["bias"])
    sigmoid, normal = torch.sigmoid(z), torch.special.ndtr(z)
    f, df = {
        "none": (z, torch.ones_like(z)),
        "relu": (torch.relu(z), torch.heaviside(z, torch.zeros_like(z))),
        "silu": (z * sigmoid, sigmoid + z * sigmoid * (1.0 - sigmoid)),
        "gelu": (z * normal, normal + z * torch.exp(-z.square() / 2.0) * (2.0 * math.pi) ** -0.5),
    }[case["act"]]
    out = {"y": f if s["residual"] is None else f + s["residual"]}
    if case["train"]:
        gz = s["grad"] * df
        out["dx"], out["dw"] = torch.mm(gz, s["weight"]), torch.mm(gz.t(), s["x"])
        if s["bias"] is not None:
            out["db"] = gz.sum(0)
        if s["residual"] is not None:
            out["dr"] = s["grad"]
    return out
