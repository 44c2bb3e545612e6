"""The training operators of a move-sequence policy, measured one call at a time.

``listed`` and ``draw`` give the cases, ``prepare`` makes a case's inputs on
the GPU, ``run`` makes one call: with ``own`` set, of this package's operators
(``alphazero_b200.ops``), otherwise of their plain form in elementary torch
operations in 32 bits.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# Work of the largest listed case; draw() stays below it.
MAX_FLOPS = 6.7e12
MAX_BYTES = 1.2e9


def listed():
    return [
        # The tokens of one move being played out in 16 games at once: latency.
        dict(name="embed_step_b19", op="embed", dtype="bf16", n=16, vocab=362, dim=256),
        # The moves of a training batch of long sequences over a large vocabulary.
        dict(name="embed_large", op="embed", dtype="bf16", n=131072, vocab=65536, dim=1024),
        # Gradient of a 19x19 move table: few rows, each met hundreds of times.
        dict(name="embed_grad_moves", op="embed_grad", dtype="fp32", n=65536, vocab=362, dim=256),
        # Gradient of a large table, a ragged number of tokens, most rows rare.
        dict(name="embed_grad_large", op="embed_grad", dtype="bf16", n=100003, vocab=65536, dim=1000),
        # One token through a wide layer: serving, bound by reading the weights.
        dict(name="linear_one_token", op="linear", dtype="bf16", m=1, k=2048, n=8192,
             act="silu", bias=True, residual=False, keep=False),
        # A pointwise layer over every point of 512 boards of 19x19 (bandwidth).
        dict(name="linear_points_b19", op="linear", dtype="bf16", m=184832, k=256, n=256,
             act="relu", bias=True, residual=True, keep=False),
        # A training batch through a wide layer that keeps z for its backward pass.
        dict(name="linear_wide", op="linear", dtype="fp16", m=16384, k=4096, n=4096,
             act="gelu", bias=True, residual=True, keep=True),
        # Its backward pass.
        dict(name="linear_grad_wide", op="linear_grad", dtype="bf16", m=8192, k=2048, n=8192,
             act="gelu", bias=True),
        # A small layer of odd sizes: a last batch, heads that fill no tile.
        dict(name="linear_grad_odd", op="linear_grad", dtype="fp16", m=4099, k=722, n=362,
             act="relu", bias=True),
        # Scoring a few continuations over a large vocabulary: reads the weights once.
        dict(name="lce_score_few", op="lce", dtype="bf16", n=13, dim=2048, vocab=65536,
             bias=False, banned=0),
        # The 19x19 move head on a training batch (361 points and pass).
        dict(name="lce_grad_moves", op="lce_grad", dtype="bf16", n=32768, dim=256, vocab=362,
             bias=True, banned=0),
        # A large vocabulary whose last entries are padding that no row may choose.
        dict(name="lce_grad_large", op="lce_grad", dtype="bf16", n=8192, dim=2048, vocab=65544,
             bias=True, banned=7),
    ]


def _log_int(rng, low, high, step=1):
    v = int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))
    v = min(high, max(low, v))
    if step > 1:
        v = max(step, v // step * step)
    return v + step if v == 3072 else v


def draw(rng):
    while True:
        op = rng.choice(["embed", "embed_grad", "linear", "linear_grad", "lce", "lce_grad"])
        half = rng.choice(["bf16", "fp16"])
        step = rng.choice([1, 8, 64])  # odd widths, aligned ones, whole tiles
        if op in ("embed", "embed_grad"):
            c = dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]), n=_log_int(rng, 1, 262144),
                     vocab=_log_int(rng, 82, 131072), dim=_log_int(rng, 32, 4096, step))
        elif op in ("linear", "linear_grad"):
            c = dict(op=op, dtype=half, m=_log_int(rng, 1, 131072), k=_log_int(rng, 32, 8192, step),
                     n=_log_int(rng, 32, 16384, step),
                     act=rng.choice(["none", "relu", "silu", "gelu"]), bias=rng.random() < 0.75)
            if op == "linear":
                c.update(residual=rng.random() < 0.5, keep=rng.random() < 0.5)
        else:
            c = dict(op=op, dtype=half, n=_log_int(rng, 1, 16384), dim=_log_int(rng, 64, 4096, step),
                     vocab=_log_int(rng, 82, 131072), bias=rng.random() < 0.5, banned=0)
            if c["bias"] and rng.random() < 0.5:
                c["banned"] = rng.randint(1, 40)
            if c["n"] * c["vocab"] > 2 ** 29:
                continue
        w = work(c)
        if w["flops"] <= MAX_FLOPS and w["bytes"] <= MAX_BYTES:
            return c


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op in ("embed", "embed_grad"):
        n, v, d = case["n"], case["vocab"], case["dim"]
        rows = min(n, v) if op == "embed" else v
        return {"bytes": 8 * n + (n + rows) * d * e, "flops": n * d}
    if op in ("linear", "linear_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        b = n if case["bias"] else 0
        if op == "linear":
            extra = m * n * (int(case["residual"]) + int(case["keep"]))
            return {"bytes": e * (m * k + n * k + m * n + b + extra), "flops": 2 * m * n * k}
        z = 0 if case["act"] == "none" else m * n
        return {"bytes": e * (2 * m * k + 2 * n * k + m * n + z + b), "flops": 4 * m * n * k}
    n, d, v = case["n"], case["dim"], case["vocab"]
    b = v if case["bias"] else 0
    if op == "lce":
        return {"bytes": e * (n * d + v * d + b) + 12 * n + 4, "flops": 2 * n * v * d}
    return {"bytes": e * 2 * (n * d + v * d + b) + 12 * n + 4, "flops": 6 * n * v * d}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 2654435761 % (2 ** 40) + 17)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dt)

    def tokens(n, vocab):  # common ones often, rare ones seldom; 3 in 100 are padding or not counted
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        t = (u * u * u * vocab).long().clamp_(max=vocab - 1)
        return torch.where(torch.rand(n, generator=g, device="cuda") < 0.03, torch.full_like(t, -1), t)

    s = dict(case)
    op = case["op"]
    if op == "embed":
        s["scale"] = math.sqrt(case["dim"])
        s["tokens"] = tokens(case["n"], case["vocab"])
        s["table"] = normal(case["vocab"], case["dim"], scale=case["dim"] ** -0.5)
    elif op == "embed_grad":
        s["scale"] = math.sqrt(case["dim"])
        s["tokens"] = tokens(case["n"], case["vocab"])
        s["grad"] = normal(case["n"], case["dim"], scale=0.01)
    elif op in ("linear", "linear_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        s["x"] = normal(m, k)
        s["weight"] = normal(n, k, scale=k ** -0.5)
        if op == "linear":
            s["b"] = normal(n, scale=0.1) if case["bias"] else None
            s["r"] = normal(m, n) if case["residual"] else None
            s["residual_scale"] = 0.5
        else:
            s["grad"] = normal(m, n, scale=0.1)
            s["z"] = None if case["act"] == "none" else normal(m, n)
    else:
        n, d, v = case["n"], case["dim"], case["vocab"]
        s["x"] = normal(n, d)
        s["weight"] = normal(v, d, scale=2.0 * d ** -0.5)
        s["targets"] = tokens(n, v - case["banned"])
        s["b"] = normal(v, scale=0.5) if case["bias"] else None
        if case["banned"]:
            s["b"][v - case["banned"]:] = -math.inf
        # half types train with a scaled loss, so that small gradients keep their bits
        s["grad_scale"] = 4096.0 if case["dtype"] == "fp16" else 1.0
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from alphazero_b200 import ops

    op = s["op"]
    if op == "embed":
        return ops.embed(s["tokens"], s["table"], scale=s["scale"])
    if op == "embed_grad":
        return ops.embed_backward(s["grad"], s["tokens"], s["vocab"], scale=s["scale"])
    if op == "linear":
        return ops.linear(s["x"], s["weight"], bias=s["b"], residual=s["r"], activation=s["act"],
                          residual_scale=s["residual_scale"], keep_preactivation=s["keep"])
    if op == "linear_grad":
        return ops.linear_backward(s["grad"], s["x"], s["weight"], preactivation=s["z"],
                                   activation=s["act"], bias=s["bias"])
    if op == "lce":
        return ops.linear_cross_entropy(s["x"], s["weight"], s["targets"], bias=s["b"])
    return ops.linear_cross_entropy_grad(s["x"], s["weight"], s["targets"], bias=s["b"],
                                         grad_scale=s["grad_scale"])


def _activate(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5


def _run_plain(s):
    op = s["op"]
    if op == "embed":
        t, table = s["tokens"], s["table"]
        y = table[t.clamp(min=0)].float() * s["scale"]
        return (y * (t >= 0)[:, None]).to(table.dtype)
    if op == "embed_grad":
        t, g = s["tokens"], s["grad"].float() * s["scale"]
        d = torch.zeros(s["vocab"], g.shape[1], device=g.device)
        d.index_add_(0, t.clamp(min=0), g * (t >= 0)[:, None])
        return d.to(s["grad"].dtype)
    x, w = s["x"].float(), s["weight"].float()
    dt = s["x"].dtype
    if op == "linear":
        z = x @ w.t()
        if s["b"] is not None:
            z = z + s["b"].float()
        y = _activate(z, s["act"])
        if s["r"] is not None:
            y = y + s["residual_scale"] * s["r"].float()
        return (y.to(dt), z.to(dt)) if s["keep"] else y.to(dt)
    if op == "linear_grad":
        g = s["grad"].float()
        if s["z"] is not None:
            g = g * _slope(s["z"].float(), s["act"])
        db = g.sum(0).to(dt) if s["bias"] else None
        return (g @ w).to(dt), (g.t() @ x).to(dt), db
    t = s["targets"]
    counted = t >= 0
    at = t.clamp(min=0)[:, None]
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    rows = (top + torch.log(total) - z.gather(1, at))[:, 0] * counted
    number = counted.sum().clamp(min=1)
    loss = rows.sum() / number
    if op == "lce":
        return loss, rows
    d = e / total
    d.scatter_add_(1, at, torch.full_like(top, -1.0))
    d *= (counted * s["grad_scale"] / number).float()[:, None]
    db = d.sum(0).to(dt) if s["b"] is not None else None
    return loss, rows, (d @ w).to(dt), (d.t() @ x).to(dt), db


def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    op = case["op"]
    if op == "embed":
        table = torch.cat([s["table"].to(f64) * s["scale"], torch.zeros(1, case["dim"], device="cuda", dtype=f64)])
        return table.index_select(0, torch.where(s["tokens"] < 0, case["vocab"], s["tokens"]))
    if op == "embed_grad":
        d = torch.zeros(case["vocab"] + 1, case["dim"], device="cuda", dtype=f64)
        d.index_add_(0, torch.where(s["tokens"] < 0, case["vocab"], s["tokens"]), s["grad"].to(f64))
        return d[:-1] * s["scale"]
    x, w = s["x"].to(f64), s["weight"].to(f64)
    if op == "linear":
        z = torch.matmul(x, w.T)
        if case["bias"]:
            z += s["b"].to(f64)
        if case["act"] == "relu":
            y = torch.relu(z)
        elif case["act"] == "silu":
            y = z * torch.sigmoid(z)
        elif case["act"] == "gelu":
            y = z * torch.special.ndtr(z)
        else:
            y = z
        if case["residual"]:
            y = y + s["residual_scale"] * s["r"].to(f64)
        return (y, z) if case["keep"] else y
    if op == "linear_grad":
        g = s["grad"].to(f64)
        if case["act"] != "none":
            z = s["z"].to(f64)
            if case["act"] == "relu":
                g = torch.where(z > 0, g, torch.zeros_like(g))
            elif case["act"] == "silu":
                p = torch.sigmoid(z)
                g = g * (p + z * p * (1 - p))
            else:
                density = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
                g = g * (torch.special.ndtr(z) + z * density)
        return torch.matmul(g, w), torch.matmul(g.T, x), g.sum(dim=0) if case["bias"] else None
    z = torch.matmul(x, w.T)
    if case["bias"]:
        z += s["b"].to(f64)
    z -= torch.logsumexp(z, dim=1, keepdim=True)
    row = torch.nonzero(s["targets"] >= 0)[:, 0]
    target = s["targets"][row]
    rows = torch.zeros(case["n"], device="cuda", dtype=f64)
    rows[row] = -z[row, target]
    count = max(1, int(row.numel()))
    if op == "lce":
        return rows.sum() / count, rows
    p = torch.exp_(z)
    p[row, target] -= 1
    p[s["targets"] < 0] = 0
    p *= s["grad_scale"] / count
    db = p.sum(dim=0) if case["bias"] else None
    return rows.sum() / count, rows, torch.matmul(p, w), torch.matmul(p.T, x), db
