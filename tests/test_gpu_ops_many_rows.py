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
