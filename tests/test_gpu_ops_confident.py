"""Rows whose target has nearly all of the probability, at logits of any size:
what is left to learn, 1 - p, is the difference of numbers that 32 bits hold to
far less of it than of themselves."""
import math

import pytest
import torch

from alphazero_b200 import ops

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("base", [0.0, 200.0, 2000.0, -2000.0])
# whole rows in TMEM, tiles, few rows by either kernel
@pytest.mark.parametrize("n,vocab,dim", [(200, 300, 8), (200, 700, 8), (3000, 2000, 64), (5, 700, 8), (13, 20003, 512)])
def test_confident_rows_at_large_logits(dtype, base, n, vocab, dim):
    # logits are exact: one product of numbers that the type holds (the target's is base + 8,
    # another's base, the rest 300 below)
    x = torch.zeros(n, dim, dtype=dtype, device="cuda")
    x[:, 0] = 1.0
    w = torch.zeros(vocab, dim, dtype=dtype, device="cuda")
    c = vocab // 2
    w[:, 0] = base - 304.0
    w[c, 0], w[c + 1, 0] = base + 8.0, base
    t = torch.full((n,), c, device="cuda")
    b = torch.zeros(vocab, dtype=dtype, device="cuda")
    scale = 4096.0 if dtype == torch.float16 else 1.0
    left = math.exp(-8) / (1 + math.exp(-8))  # 1 - p
    want = math.log1p(math.exp(-8))
    # the exponentials are good to 2^-22 of themselves and summed to 1 in 32 bits, the
    # logarithm near 1 to 2^-23
    off = 2.0 ** -21
    for loss, rows in (ops.linear_cross_entropy(x, w, t, b), ops.linear_cross_entropy_grad(x, w, t, b, scale)[:2]):
        assert (rows.double() - want).abs().max() <= off
        assert abs(loss.double().item() - want) <= off + 2.0 ** -20 * want
    _, _, _, dw, db = ops.linear_cross_entropy_grad(x, w, t, b, scale)
    # d is -left and left in two classes: off as above (the smaller probability to 2^-13 of
    # itself between two kernels), rounded once, summed over equal rows, rounded again
    # by up to the type's unit roundoff each
    for got in (dw[:, 0], db):
        for v, d in ((c, -left), (c + 1, left)):
            room = off + 2.0 ** -13 * left + 2 * UNIT[dtype] * left
            assert abs(got[v].double().item() / scale - d) <= room
        rest = torch.ones(vocab, dtype=torch.bool, device="cuda")
        rest[c:c + 2] = False
        assert not got[rest].any()


@pytest.mark.parametrize("n", [40000, 1060000])
def test_column_sums_of_confident_rows(n):
    """db of a class that every row has nearly all of its probability in."""
    vocab = 510
    x = torch.zeros(n, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(vocab, 8, dtype=torch.bfloat16, device="cuda")
    for gap in (5.0, 8.0, 9.0):
        b = torch.full((vocab,), -300.0, dtype=torch.bfloat16, device="cuda")
        b[3], b[400] = gap, 0.0
        t = torch.full((n,), 3, device="cuda")
        db = ops.linear_cross_entropy_grad(x, w, t, b)[4].double()
        left = math.exp(-gap) / (1 + math.exp(-gap))
        # each p is off by at most 2^-21 as above; sums of equal numbers at most a unit of
        # 2^-24 per addition, of which a column has fewer than 4096 in a row
        room = 2.0 ** -21 + (2.0 ** -12 + 2.0 ** -8) * left
        assert abs(db[3].item() + left) <= room and abs(db[400].item() - left) <= room
