"""The training operators on the GPU against their definitions in 64 bits
(tests/ops_reference.py holds the bounds and where they come from)."""
import math

import pytest
import torch

import ops_reference as ref
from alphazero_b200 import ops

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]
ALL = HALF + [torch.float32]
INF = math.inf


def make(*shape, dtype=torch.bfloat16, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000 + len(shape) + shape[0])
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def integers(n, low, high, seed=0, dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * n)
    return torch.randint(low, high, (n,), generator=g, device="cuda").to(dtype)


def laid(t, how):
    """t's values in another layout."""
    if how == "plain":
        return t
    if how == "transposed":
        return t.t().contiguous().t()
    if how == "offset":  # rows start anywhere, one element past an aligned address
        wide = torch.full((t.shape[0], t.shape[1] + 3), 7.0, dtype=t.dtype, device=t.device)
        wide[:, 1:1 + t.shape[1]] = t
        return wide[:, 1:1 + t.shape[1]]
    if how == "spread":  # no unit stride
        wide = torch.full((t.shape[0], 2 * t.shape[1]), 7.0, dtype=t.dtype, device=t.device)
        wide[:, ::2] = t
        return wide[:, ::2]
    raise AssertionError(how)


# ---- embedding ----

@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,vocab,dim", [(0, 5, 8), (1, 1, 1), (1, 362, 256), (7, 82, 33), (16, 362, 256),
                                         (1000, 362, 130), (513, 4000, 1024), (300, 9, 1030), (129, 20, 8200)])
def test_embed(dtype, n, vocab, dim):
    table = make(vocab, dim, dtype=dtype)
    t = integers(n, -2, vocab + 2)
    scale = 1.7
    got = ops.embed(t, table, scale)
    inside = (t >= 0) & (t < vocab)
    want = torch.where(inside[:, None], table.double()[t.clamp(0, vocab - 1)] * scale, 0.0)
    ref.within(got, want, ref.rounded(want, dtype) + 2.0 ** -23 * want.abs())


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("how", ["transposed", "offset", "spread"])
def test_embed_layouts(dtype, how):
    table = make(50, 72, dtype=dtype)
    t = integers(120, 0, 50, dtype=torch.int32)
    assert torch.equal(ops.embed(t, laid(table, how)), ops.embed(t.long(), table))
    assert torch.equal(ops.embed(t[::3], table), table[t[::3].long()])
    shaped = ops.embed(t.view(4, 5, 6), table)
    assert shaped.shape == (4, 5, 6, 72) and torch.equal(shaped.view(120, 72), table[t.long()])


def test_embed_keeps_odd_values():
    table = make(4, 40, dtype=torch.float16)
    table[1], table[2], table[3, 5] = INF, math.nan, -INF
    t = torch.tensor([0, 1, 2, 3, -1, 4, 2 ** 40], device="cuda")
    got = ops.embed(t, table, 1.0)
    assert torch.isfinite(got[0]).all() and (got[1] == INF).all() and torch.isnan(got[2]).all()
    assert got[3, 5] == -INF and (got[4:] == 0).all()


def test_embed_past_32_bits():
    vocab, dim = (1 << 20) + 3, 2056  # 2.2e9 elements
    table = torch.zeros(vocab, dim, dtype=torch.float16, device="cuda")
    table[-1], table[-2] = 3.0, 2.0
    t = torch.tensor([vocab - 1, 0, vocab - 2], device="cuda")
    assert ops.embed(t, table).float().mean(1).tolist() == [3.0, 0.0, 2.0]
    del table
    d = ops.embed_backward(torch.ones(3, dim, dtype=torch.float16, device="cuda"), t, vocab)
    assert (d[-1] == 1).all() and (d[-2] == 1).all() and (d[0] == 1).all() and not d[1:-2].any()


TOKENS = {
    "mixed": lambda n, vocab: integers(n, -1, vocab + 1),
    "one": lambda n, vocab: torch.full((n,), vocab - 1, device="cuda"),
    "none": lambda n, vocab: torch.full((n,), -1, device="cuda"),
    "skewed": lambda n, vocab: (integers(n, 0, 1000).double() / 1000).pow(4).mul(vocab).long(),
    "rising": lambda n, vocab: torch.arange(n, device="cuda") % vocab,
}


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("kind", sorted(TOKENS))
@pytest.mark.parametrize("n,vocab,dim", [(0, 5, 8), (1, 1, 1), (1, 362, 256), (33, 82, 33), (1000, 362, 130),
                                         (5000, 3, 64), (4097, 4000, 1024), (700, 70001, 20), (20011, 513, 257)])
def test_embed_backward(dtype, kind, n, vocab, dim):
    t = TOKENS[kind](n, vocab)
    g = make(n, dim, dtype=dtype) if n else torch.empty(0, dim, dtype=dtype, device="cuda")
    scale = 0.6
    got = ops.embed_backward(g, t, vocab, scale)
    at = torch.where((t >= 0) & (t < vocab), t, vocab)
    want = torch.zeros(vocab + 1, dim, dtype=torch.float64, device="cuda").index_add_(0, at, g.double())[:-1]
    size = torch.zeros(vocab + 1, dim, dtype=torch.float64, device="cuda").index_add_(0, at, g.double().abs())[:-1]
    most = int(torch.bincount(at, minlength=1).max()) if n else 0
    want = want * scale
    ref.within(got, want, ref.rounded(want, dtype) + ref.gamma(most) * scale * size)
    assert torch.equal(got, ops.embed_backward(g, t, vocab, scale))  # no order of blocks in the result


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("kind", sorted(TOKENS))
@pytest.mark.parametrize("n,vocab,dim", [(17, 1023, 65), (2000, 82, 130), (9000, 362, 64), (33000, 31, 3),
                                         (70001, 170, 258), (40000, 1000, 33), (12000, 1, 70), (1200000, 82, 40)])
def test_embed_backward_few_entries(dtype, kind, n, vocab, dim):
    test_embed_backward(dtype, kind, n, vocab, dim)


@pytest.mark.parametrize("n,vocab,dim", [(5000, 82, 48), (9000, 362, 7), (20000, 1100, 72)])
def test_embed_backward_alignment(n, vocab, dim):
    t = integers(n, -1, vocab)
    g = make(n, dim, dtype=torch.float16)
    want = ops.embed_backward(g, t, vocab)
    for how in ("transposed", "offset", "spread"):
        assert torch.equal(ops.embed_backward(laid(g, how), t, vocab), want)
    assert torch.equal(ops.embed_backward(g, t.int(), vocab), want)
    wide = torch.zeros(n, 2, dtype=torch.int64, device="cuda")
    wide[:, 0] = t
    assert torch.equal(ops.embed_backward(g, wide[:, 0], vocab), want)


def test_embed_backward_layouts():
    t = integers(240, -1, 41)
    g = make(240, 48, dtype=torch.float32)
    want = ops.embed_backward(g, t, 40)
    for how in ("transposed", "offset", "spread"):
        assert torch.equal(ops.embed_backward(laid(g, how), t, 40), want)
    assert torch.equal(ops.embed_backward(g, t.int(), 40), want)
    assert torch.equal(ops.embed_backward(g.view(6, 40, 48), t.view(6, 40), 40), want)
    row = make(1, 48, dtype=torch.float32)
    assert torch.equal(ops.embed_backward(row.expand(240, 48), t, 40),
                       ops.embed_backward(row.repeat(240, 1), t, 40))


def test_embed_gradient_by_differences():
    table = make(30, 24, dtype=torch.float32).double()
    t = integers(100, -1, 31)
    g = make(100, 24, dtype=torch.float32, seed=1)
    d = ops.embed_backward(g, t, 30, 1.3).double()
    way = make(30, 24, dtype=torch.float32, seed=2).double()

    def f(tab):  # linear in the table: a difference of any width is exact but for rounding
        y = torch.where(((t >= 0) & (t < 30))[:, None], tab[t.clamp(0, 29)] * 1.3, 0.0)
        return (y * g.double()).sum()

    slope = (f(table + way) - f(table - way)) / 2
    assert abs(slope - (d * way).sum()) <= 1e-5 * (d.abs() * way.abs()).sum()


# ---- linear layer ----

SIZES = [(1, 1, 1), (1, 16, 8), (3, 362, 722), (5, 33, 17), (64, 64, 64), (129, 257, 65), (300, 128, 1024),
         (2, 1000, 362), (16, 96, 4096), (257, 72, 40), (1000, 520, 200), (33, 8, 2050)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("name", sorted(ops.ACTIVATIONS))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear(dtype, name, m, n, k):
    x, w = make(m, k, dtype=dtype), make(n, k, dtype=dtype, seed=1, scale=k ** -0.5)
    b = make(n, dtype=dtype, seed=2) if m % 2 else None
    r = make(m, n, dtype=dtype, seed=3) if n % 2 == 0 else None
    keep = k % 2 == 0
    got = ops.linear(x, w, b, r, name, 0.5, keep)
    y, z = got if keep else (got, None)
    want, want_z, off, off_z = ref.linear(x, w, b, r, name, 0.5)
    ref.within(y, want, off)
    if keep:
        ref.within(z, want_z, off_z)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("name", sorted(ops.ACTIVATIONS))
@pytest.mark.parametrize("m,n,k", [(9, 2050, 64), (13, 5001, 72), (16, 20000, 136), (12, 40000, 7), (10, 19072, 1500),
                                   (16, 20003, 1736), (9, 65537, 520), (12, 9472, 3545), (13, 33000, 1024)])
def test_linear_few_tokens(dtype, name, m, n, k):
    test_linear(dtype, name, m, n, k)


@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("how", ["transposed", "offset", "spread"])
def test_linear_layouts(m, how):
    n, k = 136, 72
    x, w, r = make(m, k), make(n, k, seed=1, scale=0.1), make(m, n, seed=3)
    b = make(n, seed=2)
    want, want_z, off, off_z = ref.linear(x, w, b, r, "gelu", 2.0)
    for args in ((laid(x, how), w, b, r), (x, laid(w, how), b, r), (x, w, b, laid(r, how)),
                 (laid(x, how), laid(w, how), torch.stack([b, b], 1)[:, 0], laid(r, how))):
        y, z = ops.linear(*args, "gelu", 2.0, True)
        ref.within(y, want, off)
        ref.within(z, want_z, off_z)
    y = ops.linear(x[:1].expand(m, k), w, b, r[:1].expand(m, n))
    want, _, off, _ = ref.linear(x[:1].expand(m, k), w, b, r[:1].expand(m, n), "none", 1.0)
    ref.within(y, want, off)


def test_linear_shapes_and_empty():
    w = make(40, 24)
    assert ops.linear(make(2, 3, 24), w).shape == (2, 3, 40)
    assert ops.linear(make(24), w).shape == (40,)
    y, z = ops.linear(torch.empty(0, 24, dtype=torch.bfloat16, device="cuda"), w, keep_preactivation=True)
    assert y.shape == z.shape == (0, 40)
    e = torch.empty(0, 40, dtype=torch.bfloat16, device="cuda")
    dx, dw, db = ops.linear_backward(e, torch.empty(0, 24, dtype=torch.bfloat16, device="cuda"), w, e, "relu")
    assert dx.shape == (0, 24) and not dw.any() and not db.any() and dw.shape == (40, 24)


@pytest.mark.parametrize("m,n,k", [(4, 40, 64), (200, 264, 128)])
def test_linear_keeps_odd_values_to_their_rows(m, n, k):
    x, w, b = make(m, k), make(n, k, seed=1, scale=0.1), make(n, seed=2)
    good = ops.linear(x, w, b, activation="relu")
    bad = x.clone()
    bad[1, 3], bad[2, 5] = math.nan, INF
    y = ops.linear(bad, w, b, activation="relu")
    same = torch.ones(m, dtype=torch.bool, device="cuda")
    same[1:3] = False
    assert torch.equal(y[same], good[same]) and torch.isnan(y[1]).all()
    assert not torch.isfinite(y[2][w[:, 5] > 0]).any() and (y[2][w[:, 5] < 0] == 0).all()
    b[7] = -INF
    y, z = ops.linear(x, w, b, activation="relu", keep_preactivation=True)
    assert (z[:, 7] == -INF).all() and (y[:, 7] == 0).all() and torch.isfinite(y).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("name", sorted(ops.ACTIVATIONS))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_backward(dtype, name, m, n, k):
    g, x = make(m, n, dtype=dtype, seed=4), make(m, k, dtype=dtype)
    w, z = make(n, k, dtype=dtype, seed=1, scale=k ** -0.5), make(m, n, dtype=dtype, seed=5)
    z[0, 0] = 0.0
    bias = k % 3 != 0
    got = ops.linear_backward(g, x, w, z, name, bias)
    want = ref.linear_backward(g, x, w, z, name)
    for a, (b, off) in list(zip(got, want))[:3 if bias else 2]:
        ref.within(a, b, off)
    assert bias or got[2] is None
    for a, b in zip(got, ops.linear_backward(g, x, w, z, name, bias)):
        assert a is None or torch.equal(a, b)


@pytest.mark.parametrize("m", [3, 300])
@pytest.mark.parametrize("name", ["none", "silu"])
@pytest.mark.parametrize("how", ["transposed", "offset", "spread"])
def test_linear_backward_layouts(m, name, how):
    n, k = 136, 72
    g, x, w, z = make(m, n), make(m, k, seed=1), make(n, k, seed=2, scale=0.1), make(m, n, seed=3)
    want = ref.linear_backward(g, x, w, z, name)
    for args in ((laid(g, how), x, w, z), (g, laid(x, how), w, z), (g, x, laid(w, how), z),
                 (g, x, w, laid(z, how))):
        for a, (b, off) in zip(ops.linear_backward(*args, name), want):
            ref.within(a, b, off)
    one = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(m, n)  # the gradient of a sum
    for a, (b, off) in zip(ops.linear_backward(one, x, w, z, name), ref.linear_backward(one, x, w, z, name)):
        ref.within(a, b, off)


@pytest.mark.parametrize("name", ["none", "silu", "gelu"])
def test_linear_gradient_by_differences(name):
    m, n, k = 70, 48, 40
    x, w, b = (make(m, k, dtype=torch.float16), make(n, k, dtype=torch.float16, seed=1, scale=0.2),
               make(n, dtype=torch.float16, seed=2))
    g = make(m, n, dtype=torch.float16, seed=3)
    # a kept z that is exactly the 64-bit one, so that the differences are of the same function
    z = (x.double() @ w.double().t() + b.double())
    got = ops.linear_backward(g, x, w, z.half(), name)
    h = 1e-5
    for at, d in enumerate(got):
        way = make(*d.shape, dtype=torch.float32, seed=7 + at).double()

        def f(s):
            p = [t.double() for t in (x, w, b)]
            p[at] = p[at] + s * way
            return (ref.act(p[0] @ p[1].t() + p[2], name) * g.double()).sum()

        slope = (f(h) - f(-h)) / (2 * h)
        # z, g and d are rounded to 11 bits, each independently of the direction
        assert abs(slope - (d.double() * way).sum()) <= 4 * 2.0 ** -11 * (d.double() * way).norm() * 8 + 1e-6


# ---- linear cross entropy ----

def check_cross_entropy(x, w, t, b=None, grad_scale=1.0):
    got = ops.linear_cross_entropy_grad(x, w, t, b, grad_scale)
    want = ref.cross_entropy(x, w, b, t.long(), grad_scale)
    for a, (v, off) in zip(got, want):
        if a is not None:
            ref.within(a, v, off)
    assert (got[4] is None) == (b is None)
    loss, rows = ops.linear_cross_entropy(x, w, t, b)
    ref.within(loss, *want[0])
    ref.within(rows, *want[1])
    for a, c in zip(got, ops.linear_cross_entropy_grad(x, w, t, b, grad_scale)):
        assert a is None or torch.equal(a, c)
    return got


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,vocab,dim", [(1, 1, 1), (1, 362, 256), (3, 2, 8), (5, 82, 33), (130, 362, 64),
                                         (300, 1000, 40), (64, 128, 128), (257, 129, 72), (13, 5000, 520),
                                         (1000, 83, 1030)])
def test_cross_entropy(dtype, bias, n, vocab, dim):
    x, w = make(n, dim, dtype=dtype), make(vocab, dim, dtype=dtype, seed=1, scale=2 * dim ** -0.5)
    b = make(vocab, dtype=dtype, seed=2) if bias else None
    check_cross_entropy(x, w, integers(n, -1, vocab + 1), b, 512.0 if dtype == torch.float16 else 1.0)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n,vocab,dim", [(17, 1, 64), (100, 64, 70), (255, 65, 8), (256, 82, 256), (258, 128, 64),
                                         (700, 170, 128), (1030, 256, 33), (513, 257, 64), (300, 362, 4000),
                                         (40, 384, 64), (333, 385, 72), (129, 448, 128), (600, 512, 64),
                                         (31, 513, 64), (19500, 362, 64), (40000, 82, 40)])
def test_cross_entropy_few_classes(bias, n, vocab, dim):
    x, w = make(n, dim), make(vocab, dim, seed=1, scale=2 * dim ** -0.5)
    b = make(vocab, seed=2) if bias else None
    check_cross_entropy(x, w, integers(n, -1, vocab + 1), b)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,vocab,dim", [(16, 20003, 264), (9, 2048, 64), (10, 2049, 65), (12, 19001, 1030), (16, 20003, 1736),
                                         (11, 65537, 520)])
def test_cross_entropy_few_rows(dtype, n, vocab, dim):
    x, w = make(n, dim, dtype=dtype), make(vocab, dim, dtype=dtype, seed=1, scale=2 * dim ** -0.5)
    b = make(vocab, dtype=dtype, seed=2)
    b[vocab // 2:vocab // 2 + 200] = -INF
    check_cross_entropy(x, w, integers(n, -1, vocab // 2), b, 512.0 if dtype == torch.float16 else 1.0)


@pytest.mark.parametrize("low", [-INF, -3.0e38])
def test_cross_entropy_few_classes_banned(low):
    n, vocab = 200, 450
    x, w, b = make(n, 64), make(vocab, 64, seed=1, scale=0.3), make(vocab, seed=2)
    b[64:450] = low  # whole halves of a row among them
    t = integers(n, 0, 64)
    got = check_cross_entropy(x, w, t, b)
    assert not got[3][64:].any() and not got[4][64:].any()
    b[:] = low
    got = check_cross_entropy(x, w, t, b)
    if low == -INF:
        assert (got[1] == INF).all()
    assert torch.isfinite(got[2]).all() and torch.isfinite(got[3]).all()


@pytest.mark.parametrize("how", ["transposed", "offset", "spread"])
def test_cross_entropy_layouts(how):
    x, w, b = make(150, 72), make(390, 72, seed=1, scale=0.2), make(390, seed=2)
    t = integers(150, -1, 390, dtype=torch.int32)
    check_cross_entropy(laid(x, how), w, t, b)
    check_cross_entropy(x, laid(w, how), t, b)
    check_cross_entropy(x[:75], w, t[::2], b)
    check_cross_entropy(x[:1].expand(150, 72), w, t, b)


def test_cross_entropy_counts():
    x, w = make(40, 64), make(200, 64, seed=1)
    b = make(200, seed=2)
    none = torch.full((40,), -1, device="cuda")
    got = check_cross_entropy(x, w, none, b)
    assert got[0] == 0 and not any(t.any() for t in got[1:])
    one = none.clone()
    one[17] = 199
    check_cross_entropy(x, w, one, b)
    e = torch.empty(0, 64, dtype=torch.bfloat16, device="cuda")
    loss, rows, dx, dw, db = ops.linear_cross_entropy_grad(e, w, none[:0], b)
    assert loss == 0 and rows.shape == (0,) and dx.shape == (0, 64) and not dw.any() and not db.any()
    x[3] = math.nan  # a row that is not counted has no loss, whatever it holds
    one = integers(40, 0, 200)
    one[3] = -1
    loss, rows, dx, _, _ = ops.linear_cross_entropy_grad(x, w, one, b)
    assert torch.isfinite(loss) and torch.isfinite(rows).all() and torch.isfinite(dx).all()


@pytest.mark.parametrize("n", [4, 200])
@pytest.mark.parametrize("low", [-INF, -3.0e38])
def test_cross_entropy_banned(n, low):
    vocab = 700
    x, w, b = make(n, 64), make(vocab, 64, seed=1, scale=0.3), make(vocab, seed=2)
    b[256:600] = low
    t = integers(n, 0, 256)
    got = check_cross_entropy(x, w, t, b)
    assert not got[3][256:600].any() and not got[4][256:600].any()
    if low == -INF:
        t[1] = 300  # a banned target: probability 0
        got = check_cross_entropy(x, w, t, b)
        assert got[1][1] == INF and got[0] == INF and torch.isfinite(got[2]).all()
        b[:] = low  # nothing is left in any row
        got = check_cross_entropy(x, w, t, b)
        assert (got[1] == INF).all() and torch.isfinite(got[2]).all() and torch.isfinite(got[3]).all()


@pytest.mark.parametrize("n", [4, 200])
def test_cross_entropy_odd_values(n):
    x, w = make(n, 64), make(300, 64, seed=1)
    t = integers(n, 0, 300)
    x[1, 0] = math.nan
    loss, rows, dx, dw, _ = ops.linear_cross_entropy_grad(x, w, t)
    assert torch.isnan(loss) and torch.isnan(rows[1]) and torch.isnan(dx[1]).all()
    other = torch.ones(n, dtype=torch.bool, device="cuda")
    other[1] = False
    assert torch.isfinite(rows[other]).all() and torch.isfinite(dx[other]).all()
    # logits in the thousands: the sums stay finite
    check_cross_entropy(make(n, 64, scale=30.0), make(300, 64, seed=1, scale=30.0), t)


def test_cross_entropy_in_several_pieces():
    n, vocab, dim = 2500, 131077, 24
    x, w, b = make(n, dim), make(vocab, dim, seed=1, scale=0.5), make(vocab, seed=2)
    check_cross_entropy(x, w, integers(n, -5, vocab), b)


def test_cross_entropy_few_classes_in_several_pieces():
    n, vocab, dim = 1060000, 510, 8
    x, w, b = make(n, dim), make(vocab, dim, seed=1, scale=0.5), make(vocab, seed=2)
    check_cross_entropy(x, w, integers(n, -1, vocab), b)


def test_autograd_once():
    x, w = make(20, 64).requires_grad_(), make(40, 64, seed=1, scale=0.2).requires_grad_()
    y = ops.linear_layer(x, w, activation="gelu")
    (d,) = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.float().sum(), w)


def test_cross_entropy_gradient_by_differences():
    n, vocab, dim = 60, 100, 32
    x, w, b = (make(n, dim, dtype=torch.float16), make(vocab, dim, dtype=torch.float16, seed=1, scale=0.3),
               make(vocab, dtype=torch.float16, seed=2))
    t = integers(n, -1, vocab)
    scale = 256.0
    got = ops.linear_cross_entropy_grad(x, w, t, b, scale)[2:]
    counted = t >= 0
    h = 1e-5
    for at, d in enumerate(got):
        way = make(*d.shape, dtype=torch.float32, seed=7 + at).double()

        def f(s):
            p = [v.double() for v in (x, w, b)]
            p[at] = p[at] + s * way
            lp = torch.log_softmax(p[0] @ p[1].t() + p[2], 1)
            return -(lp[counted].gather(1, t[counted][:, None])).sum() / counted.sum() * scale

        slope = (f(h) - f(-h)) / (2 * h)
        # d and the result are rounded to 11 bits, each independently of the direction
        assert abs(slope - (d.double() * way).sum()) <= 3 * 2.0 ** -11 * (d.double() * way).norm() * 8 + 1e-6


# ---- streams, graphs, autograd, status ----

def step(x, w, b, t, table, tokens):
    y, z = ops.linear(x, w, b, None, "gelu", 1.0, True)
    return [ops.embed(tokens, table, 2.0), y, *ops.linear_backward(y, x, w, z, "gelu"),
            ops.embed_backward(x, tokens, 500), *ops.linear_cross_entropy_grad(x, w, t, b)]


def inputs(n=260, seed=0):
    return (make(n, 64, seed=seed), make(500, 64, seed=seed + 1, scale=0.2), make(500, seed=seed + 2),
            integers(n, -1, 500, seed=seed), make(500, 64, seed=seed + 3), integers(n, -1, 500, seed=seed + 4))


def test_other_streams_and_graphs():
    a, c = inputs(), inputs(seed=20)
    want = step(*a), step(*c)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):  # two streams at once, each with its own scratch
        with torch.cuda.stream(s1):
            one = step(*a)
        with torch.cuda.stream(s2):
            two = step(*c)
        torch.cuda.synchronize()
        for got, w in ((one, want[0]), (two, want[1])):
            assert all(torch.equal(p, q) for p, q in zip(got, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*a)
    for new in (c, inputs(seed=40)):
        for to, frm in zip(a, new):
            to.copy_(frm)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(held, step(*a)))
    ops.synchronize()


def test_autograd_matches_torch():
    n, dim, vocab = 90, 64, 150
    tokens, t = integers(n, 0, 82, seed=3), integers(n, 0, vocab, seed=4)
    given = [make(82, dim, dtype=torch.float16, seed=1), make(96, dim, dtype=torch.float16, seed=2, scale=0.1),
             make(96, dtype=torch.float16, seed=3), make(n, 96, dtype=torch.float16, seed=4),
             make(vocab, 96, dtype=torch.float16, seed=5, scale=0.1), make(vocab, dtype=torch.float16, seed=6)]

    def run(p, mine):
        table, w, b, r, head, hb = p
        if mine:
            h = ops.embedding(tokens, table, 2.0)
            h = ops.linear_layer(h, w, b, r, "silu", 0.5)
            return ops.cross_entropy_loss(h, head, t, hb, grad_scale=1024.0) * 64.0
        h = torch.nn.functional.silu((table[tokens] * 2.0) @ w.t() + b) + 0.5 * r
        return torch.nn.functional.cross_entropy(h @ head.t() + hb, t) * 64.0

    mine = [p.clone().requires_grad_() for p in given]
    loss = run(mine, True)
    loss.backward()
    exact = [p.double().requires_grad_() for p in given]
    want = run(exact, False)
    want.backward()
    assert abs(loss.item() - want.item()) < 2e-3 * want.item()
    for a, b in zip(mine, exact):
        # every stage rounds to 11 bits: five roundings in the longest chain
        assert (a.grad.double() - b.grad).norm() <= 5 * 2.0 ** -11 * 2 * b.grad.norm()
