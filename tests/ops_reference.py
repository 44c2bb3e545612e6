"""The training operators in 64 bits, and how far a kernel may be from them.

Bounds are for each element, from the arithmetic the operators promise:
operands as given, products summed in 32 bits in any order, each output (and,
where the interface says so, one intermediate) rounded once to the operands'
type.  With u the type's unit roundoff and gamma(K) = (K + 8) 2^-23, a sum of
K products p_k is off by at most gamma(K) sum |p_k| (twice the classical bound
K 2^-24, since a tensor core may truncate), and a rounded value v by u |v|
plus half the smallest subnormal."""
import math

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def gamma(k):
    return (k + 8) * 2.0 ** -23


def rounded(v, dtype):
    return UNIT[dtype] * v.abs() + TINY[dtype]


def within(got, want, bound):
    """Asserts |got - want| <= bound for every element (equal where want is
    infinite, NaN where it is NaN)."""
    got = got.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd])
    # what was rounded is the computed value, which the other bound moves
    off = (got - want).abs()[fine]
    top = (bound.expand_as(want)[fine]) * (1 + 2.0 ** -6)
    worst = (off - top).max().item() if off.numel() else 0.0
    assert worst <= 0, f"an element is {worst:.3e} past its bound"


def act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return z * 0.5 * (1 + torch.erf(z / math.sqrt(2)))
    return z


def slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def linear(x, w, b, r, name, r_scale):
    """y, z and their bounds."""
    x64, w64 = x.double(), w.double()
    k = x.shape[-1]
    z = x64 @ w64.t()
    size = x64.abs() @ w64.abs().t()
    if b is not None:
        z = z + b.double()
        size = size + b.double().abs()
    off = gamma(k) * size
    y = act(z, name)
    # |act'| < 1.2; expf and erff are within a few units of 2^-24
    y_off = 1.2 * off + 2.0 ** -20 * y.abs() + (2.0 ** -21 * z.abs() if name in ("silu", "gelu") else 0)
    if r is not None:
        y = y + r_scale * r.double()
        y_off = y_off + 2.0 ** -22 * (r_scale * r.double()).abs()
    return y, z, y_off + rounded(y, x.dtype), off + rounded(z, x.dtype)


def linear_backward(g, x, w, z, name):
    """(dx, dw, db) and their bounds."""
    g64, x64, w64 = g.double(), x.double(), w.double()
    n, k, m = w.shape[0], w.shape[1], g64.shape[0]
    u = 0.0
    tiny = 0.0
    if name != "none":
        g64 = g64 * slope(z.double(), name)
        # the slope is within 2^-20 of the formula's, then g is rounded once
        u = UNIT[x.dtype] + 2.0 ** -20
        tiny = TINY[x.dtype] + 2.0 ** -20 * g.double().abs().max().item() if m else 0.0
    dx, dw, db = g64 @ w64, g64.t() @ x64, g64.sum(0)
    a = g64.abs()
    ax = (u + gamma(n)) * (a @ w64.abs()) + tiny * w64.abs().sum(0)
    aw = (u + gamma(m)) * (a.t() @ x64.abs()) + tiny * x64.abs().sum(0)
    ab = (u + gamma(m)) * a.sum(0) + tiny * m
    return ((dx, ax + rounded(dx, x.dtype)), (dw, aw + rounded(dw, x.dtype)),
            (db, ab + rounded(db, x.dtype)))


def cross_entropy(x, w, b, t, grad_scale):
    """(loss, rows, dx, dw, db), each with its bound."""
    x64, w64 = x.double(), w.double()
    n, dim = x64.shape
    vocab = w64.shape[0]
    z = x64 @ w64.t()
    size = x64.abs() @ w64.abs().t()
    if b is not None:
        z = z + b.double()
        size = size + torch.nan_to_num(b.double().abs(), posinf=0.0)
    counted = (t >= 0) & (t < vocab)
    count = max(1, int(counted.sum()))
    # a logit is off by eps, so the log of the sum is too, and expf and logf add a little
    eps = gamma(dim) * size.amax(1, keepdim=True) + 2.0 ** -20
    top = z.amax(1, keepdim=True)
    dead = top == -math.inf
    zs = torch.where(dead, torch.full_like(z, -math.inf), z - torch.where(dead, torch.zeros_like(top), top))
    total = torch.exp(zs).sum(1, keepdim=True)
    lp = torch.where(dead, torch.full_like(z, -math.inf), zs - torch.log(total))
    at = torch.where(counted, t, torch.zeros_like(t))[:, None]
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    rows = torch.where(counted, -lp.gather(1, at)[:, 0], zero)
    logit = torch.where(torch.isfinite(z.gather(1, at)[:, 0]), z.gather(1, at)[:, 0].abs(), zero)
    rows_off = 2 * eps[:, 0] + 2.0 ** -20 * (logit + torch.nan_to_num(rows.abs(), posinf=0.0))
    loss = rows.sum() / count
    loss_off = rows_off.sum() / count + (n + 8) * 2.0 ** -23 * torch.nan_to_num(rows, posinf=0.0).sum() / count
    p = torch.exp(lp)
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    d = torch.where(counted[:, None], p - hot, zero)
    u = UNIT[x.dtype]
    # probabilities are good to 2 eps and 2^-13 of their size, or 2^-27; d is rounded once
    # (float16 keeps 2^14 d, whose smallest steps are 2^-38)
    d_off = torch.where(counted[:, None], p * (2 * eps + 2.0 ** -13) + 2.0 ** -27 + u * d.abs() + 2.0 ** -38, zero)
    s = grad_scale / count
    w0, x0 = w64.abs(), x64.abs()
    dx = (d @ w64) * s
    dx_off = (d_off @ w0 + gamma(vocab) * (d.abs() @ w0)) * s
    dw = (d.t() @ x64) * s
    dw_off = (d_off.t() @ x0 + gamma(n) * (d.abs().t() @ x0)) * s
    db = d.sum(0) * s
    db_off = (d_off.sum(0) + gamma(n) * d.abs().sum(0)) * s
    dt = x.dtype
    return ((loss, loss_off), (rows, rows_off), (dx, dx_off + rounded(dx, dt)),
            (dw, dw_off + rounded(dw, dt)), (db, db_off + rounded(db, dt)))
