"""Infinities and NaN in rows that the training operators leave out, or that
an activation shuts: what has no part in a result leaves no trace in it."""
import math

import pytest
import torch

from alphazero_b200 import ops
from test_gpu_ops import integers, laid, make

pytestmark = pytest.mark.gpu

INF = math.inf


def uncounted(n, vocab, seed=0):
    """Targets of which a few, the last row's among them, are not counted."""
    t = integers(n, 0, vocab, seed=seed)
    out = torch.unique(torch.tensor([0, n // 3, n // 2, n - 1], device="cuda").clamp(min=0, max=n - 1))
    t[out] = torch.tensor([-1, vocab, 2 ** 40, -7], device="cuda")[:out.numel()]
    return t, out


# whole rows in TMEM, tiles, few rows by either kernel, several pieces of each way
SHAPES = [(40, 200, 64), (700, 362, 256), (1000, 82, 40), (129, 512, 1024), (200, 700, 64), (300, 1000, 1100),
          (4100, 520, 33), (5, 700, 264), (13, 20003, 264), (2500, 131077, 24), (1060000, 510, 8)]


@pytest.mark.parametrize("n,vocab,dim", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_uncounted_rows_leave_no_trace(dtype, n, vocab, dim):
    x, w = make(n, dim, dtype=dtype), make(vocab, dim, dtype=dtype, seed=1, scale=dim ** -0.5)
    w[:, 1], w[:, 2], w[:, 3] = -w[:, 1].abs() - 0.01, w[:, 2].abs() + 0.01, 0.0
    b = make(vocab, dtype=dtype, seed=2)
    t, out = uncounted(n, vocab)
    scale = 512.0 if dtype == torch.float16 else 1.0
    x[out] = 0.0
    want = ops.linear_cross_entropy_grad(x, w, t, b, scale)
    assert all(torch.isfinite(v).all() for v in want)
    fills = [lambda r: r.fill_(math.nan), lambda r: r[:, 0].fill_(math.nan), lambda r: r[:, 1].fill_(INF),
             lambda r: r[:, 1].fill_(-INF), lambda r: r[:, 2].fill_(INF), lambda r: r[:, 3].fill_(INF)]
    for fill in fills if n < 10000 else fills[:2]:
        rows = torch.zeros(out.numel(), dim, dtype=dtype, device="cuda")
        fill(rows)
        bad = x.clone()
        bad[out] = rows
        for a, c in zip(ops.linear_cross_entropy_grad(bad, w, t, b, scale), want):
            assert torch.equal(a, c)


@pytest.mark.parametrize("how", ["transposed", "offset", "spread"])
@pytest.mark.parametrize("n,vocab", [(150, 390), (150, 900), (64, 64), (1, 700), (70, 5000)])
def test_uncounted_rows_in_other_layouts(how, n, vocab):
    x, w, b = make(n, 72), make(vocab, 72, seed=1, scale=0.2), make(vocab, seed=2)
    t, out = uncounted(n, vocab)
    x[out] = 0.0
    want = ops.linear_cross_entropy_grad(x, w, t, b)
    x[out] = math.nan
    for a, c in zip(ops.linear_cross_entropy_grad(laid(x, how), w, t, b), want):
        assert torch.equal(a, c)


def test_only_uncounted_rows_and_all_of_them_bad():
    for vocab in (82, 900):
        x, w, b = make(300, 64), make(vocab, 64, seed=1), make(vocab, seed=2)
        x[:] = math.nan
        got = ops.linear_cross_entropy_grad(x, w, torch.full((300,), -1, device="cuda"), b)
        assert not any(v.any() for v in got)


def test_counted_rows_keep_their_nan():
    """A bad row that is counted shows in every gradient that it has a part in."""
    for vocab in (82, 900):
        x, w, b = make(300, 64), make(vocab, 64, seed=1), make(vocab, seed=2)
        t, out = uncounted(300, vocab)
        x[out] = math.nan
        x[7, 5] = math.nan
        loss, rows, dx, dw, db = ops.linear_cross_entropy_grad(x, w, t, b)
        assert torch.isnan(loss) and torch.isnan(rows[7]) and torch.isnan(dx[7]).all()
        assert torch.isnan(dw).all() and torch.isnan(db).all()  # d of row 7 is NaN in every class
        assert not dx[out].any() and not rows[out].any()


# ---- gradients of the linear layer and of the embedding ----

@pytest.mark.parametrize("n", [40, 37])  # by eight columns, one by one
@pytest.mark.parametrize("value", [INF, -INF, math.nan])
def test_a_shut_relu_lets_nothing_through(n, value):
    m, k = 70, 24
    g, x, w, z = make(m, n), make(m, k, seed=1), make(n, k, seed=2), make(m, n, seed=3)
    z[5, 3], z[6, 4], z[7, 9] = -1.0, 0.0, -INF
    want = ops.linear_backward(g, x, w, z, "relu")
    bad = g.clone()
    for i, j in ((5, 3), (6, 4), (7, 9)):
        bad[i, j] = value
    for a, b in zip(ops.linear_backward(bad, x, w, z, "relu"), want):
        assert torch.equal(a, b) and torch.isfinite(a).all()


@pytest.mark.parametrize("name", ["none", "relu", "silu", "gelu"])
def test_linear_backward_keeps_odd_values_to_their_places(name):
    m, n, k = 70, 40, 24
    g, x, w, z = make(m, n), make(m, k, seed=1), make(n, k, seed=2), make(m, n, seed=3).abs()
    good = ops.linear_backward(g, x, w, z, name)
    bad = g.clone()
    bad[9, 11] = math.nan
    dx, dw, db = ops.linear_backward(bad, x, w, z, name)
    rows, cols = torch.arange(m, device="cuda") != 9, torch.arange(n, device="cuda") != 11
    assert torch.equal(dx[rows], good[0][rows]) and torch.isnan(dx[9]).all()
    assert torch.equal(dw[cols], good[1][cols]) and torch.isnan(dw[11]).all()
    assert torch.equal(db[cols], good[2][cols]) and torch.isnan(db[11])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n", [50, 5000])
def test_embed_backward_keeps_odd_values_to_their_entries(dtype, n):
    vocab, dim = 82, 40
    t = integers(n, 0, vocab - 2)
    t[::7], t[1::7] = -1, vocab
    g = make(n, dim, dtype=dtype)
    good = ops.embed_backward(g, t, vocab)
    bad = g.clone()
    bad[::7], bad[1::7] = math.nan, INF  # padding
    assert torch.equal(ops.embed_backward(bad, t, vocab), good)
    bad[2, 3], bad[3, 4] = math.nan, -INF
    d = ops.embed_backward(bad, t, vocab)
    hit = torch.zeros(vocab, dim, dtype=torch.bool, device="cuda")
    hit[t[2], 3] = hit[t[3], 4] = True
    assert torch.isnan(d[t[2], 3]) and not torch.isfinite(d[t[3], 4])
    assert torch.equal(d[~hit], good[~hit])
