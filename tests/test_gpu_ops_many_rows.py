"""Calls of so many rows that they are taken in pieces, and sums over so many
rows that a bound on their rounding would let anything pass: rows are compared
by sample, sums with inputs whose sums are exact in 32 bits."""
import pytest
import torch

import ops_reference as ref
from alphazero_b200 import ops
from test_gpu_ops import integers, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,vocab", [(70000, 131077), (17000000, 510), (12000000, 730)])
def test_scoring_in_several_pieces(n, vocab):
    x, w, b = make(n, 8), make(vocab, 8, seed=1, scale=0.5), make(vocab, seed=2)
    t = integers(n, -1, vocab)
    loss, rows = ops.linear_cross_entropy(x, w, t, b)
    at = torch.cat([torch.arange(n // 8 * i, n // 8 * i + 40, device="cuda") for i in range(8)]
                   + [torch.arange(n - 40, n, device="cuda")])
    for part in at.split(60):
        want = ref.cross_entropy(x[part], w, b, t[part], 1.0)[1]
        ref.within(rows[part], *want)
    assert torch.isfinite(rows).all() and not rows[t < 0].any()
    mean = rows.double().sum() / (t >= 0).sum()
    # losses are positive: summed in 32 bits by blocks of at most 1024 * 1024, then those
    assert abs(loss.item() - mean.item()) <= 2.0 ** -24 * 4096 * mean.item()


def exactly(got, want, factor, dtype):
    """got is want * factor, rounded once (want a whole number that 32 bits hold, as
    every sum on the way to it is; factor a power of two)."""
    assert torch.equal(got, (want.float() * factor).to(dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["one", "two", "skewed", "mixed", "rising"])
@pytest.mark.parametrize("n,vocab,dim", [(40000, 362, 33), (70001, 170, 258), (100003, 20000, 40), (1200000, 82, 40),
                                         (300000, 5, 1032)])
def test_embed_backward_of_long_runs_is_exact(dtype, kind, n, vocab, dim):
    """Runs over hundreds and thousands of windows: a stretch that is left out or
    taken twice shows, since sums of whole numbers below 2^24 do not round."""
    t = {"one": lambda: torch.full((n,), vocab - 1, device="cuda"),
         "two": lambda: (torch.arange(n, device="cuda") >= n // 3).long() * (vocab - 1),
         "skewed": lambda: (integers(n, 0, 1000).double() / 1000).pow(4).mul(vocab).long(),
         "mixed": lambda: integers(n, -1, vocab + 1),
         "rising": lambda: torch.arange(n, device="cuda") % vocab}[kind]()
    g = integers(n * dim, -8, 12, seed=3).view(n, dim)  # mean 1.5: a lost row is a lost 1.5
    got = ops.embed_backward(g.to(dtype), t, vocab, 0.5)
    at = torch.where((t >= 0) & (t < vocab), t, vocab)
    want = torch.zeros(vocab + 1, dim, dtype=torch.int64, device="cuda").index_add_(0, at, g)[:-1]
    assert want.abs().max() < 2 ** 24
    if dtype == torch.float16:  # in range
        keep = want.abs() < 60000
        got, want = got[keep], want[keep]
    exactly(got, want, 0.5, dtype)
    count = torch.bincount(at, minlength=vocab + 1)[:-1].clamp(max=30000)
    ones = ops.embed_backward(torch.ones(n, dim, dtype=dtype, device="cuda"), t, vocab)
    exactly(ones[count < 30000], count[count < 30000, None].expand(-1, dim), 1.0, dtype)


@pytest.mark.parametrize("m", [5000, 70001, 1000003])
@pytest.mark.parametrize("name", ["none", "relu"])
def test_linear_gradients_over_many_rows_are_exact(m, name):
    n, k = 40, 24
    g, x = integers(m * n, -2, 4, seed=1).view(m, n), integers(m * k, -1, 3, seed=2).view(m, k)
    z = integers(m * n, -1, 3, seed=3).view(m, n)
    w = make(n, k)
    _, dw, db = ops.linear_backward(g.bfloat16(), x.bfloat16(), w, z.bfloat16(), name)
    live = g * (z > 0) if name == "relu" else g
    want = (live.double().t() @ x.double()).round()
    assert live.abs().sum(0).max() < 2 ** 24 and (live.abs().double().t() @ x.abs().double()).max() < 2 ** 24
    exactly(dw, want, 1.0, torch.bfloat16)
    exactly(db, live.sum(0), 1.0, torch.bfloat16)


@pytest.mark.parametrize("m", [5000, 70001, 1000003])
def test_linear_gradients_miss_no_step(m):
    """Every 64 rows have a weight of their own, and the weights sum to zero: what is
    left is the last few rows' part, exact in 8 bits, and any lost stretch is far
    larger."""
    n, k = 40, 24
    steps = (m + 63) // 64
    weight = integers(steps, -3, 3, seed=9)
    weight[weight >= 0] += 1  # none is zero
    weight[-1] = 2  # a step of m % 64 rows
    body = weight[:-1]
    while (total := int(body.sum())) != 0:
        some = torch.nonzero((body < 2) & (body != -1) if total < 0 else (body > -2) & (body != 1))[:abs(total), 0]
        body[some] += 1 if total < 0 else -1
    assert (weight != 0).all()
    per_row = weight.repeat_interleave(64)[:m]
    u, v = 1 + torch.arange(n, device="cuda") % 2, 1 - 2 * (torch.arange(k, device="cuda") % 2)
    g, x = per_row[:, None] * u, v.expand(m, k).contiguous()
    _, dw, db = ops.linear_backward(g.bfloat16(), x.bfloat16(), make(n, k))
    left = 2 * (m - 64 * (steps - 1))
    exactly(dw, left * u[:, None] * v, 1.0, torch.bfloat16)
    exactly(db, left * u, 1.0, torch.bfloat16)


@pytest.mark.parametrize("n", [5000, 70001, 1060000])
def test_cross_entropy_sums_over_many_rows(n):
    """Logits of zero over 512 classes: d is 2^-9, or 2^-9 - 1 at the target, which
    float16 holds, and sums of those times small whole numbers are whole
    multiples of 2^-9 that 32 bits hold; only the exponential's last bits and
    the scale round."""
    vocab, dim = 512, 16
    # of mean 0: a lost row changes a class's sum by a few hundredths of it
    x = integers(n * dim, -2, 3, seed=1).view(n, dim)
    t = integers(n, -1, vocab, seed=2)
    w = torch.zeros(vocab, dim, dtype=torch.float16, device="cuda")
    b = torch.zeros(vocab, dtype=torch.float16, device="cuda")
    counted = t >= 0
    count = int(counted.sum())
    # as large as float16 takes: the largest sums are of a column's mean of x, and of its targets
    scale = 64.0
    loss, rows, dx, dw, db = ops.linear_cross_entropy_grad(x.half(), w, t, b, scale)
    at = torch.where(counted, t, vocab)
    hot = torch.zeros(vocab + 1, dim, dtype=torch.int64, device="cuda").index_add_(0, at, x)[:-1]
    every = x[counted].sum(0)
    want = (every[None].double() / vocab - hot) * (scale / count)
    # 2^-21 of each p for the exponential, 2^-22 for scale and division, and one rounding
    # (sums of products by the tensor cores and of a column in 32 bits round no further)
    size = x[counted].abs().sum(0).double()[None] / vocab
    size_hot = torch.zeros(vocab + 1, dim, dtype=torch.int64, device="cuda").index_add_(0, at, x.abs())[:-1]
    off = (size * 2.0 ** -20 + size_hot * 2.0 ** -20) * (scale / count) + ref.rounded(want, torch.float16)
    assert ((dw.double() - want).abs() <= off).all()
    many = torch.bincount(at, minlength=vocab + 1)[:-1].double()
    want = (count / vocab - many) * (scale / count)
    off = (count / vocab + many) * 2.0 ** -20 * (scale / count) + ref.rounded(want, torch.float16)
    assert ((db.double() - want).abs() <= off).all()
    assert not dx.any()
    assert (rows[counted].double() - 9 * 0.6931471805599453).abs().max() <= 2.0 ** -20 * 9 and not rows[~counted].any()
    assert abs(loss.item() - 9 * 0.6931471805599453) <= 2.0 ** -18 * 9
