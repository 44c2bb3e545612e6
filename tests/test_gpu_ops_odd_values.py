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
