"""Scalars that do not fit raise ValueError or TypeError, like tensors that do
not."""
import pytest
import torch

from alphazero_b200 import ops
from test_gpu_ops import integers, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", ["2", None, 1j])
def test_scales(value):
    x, w, t = make(4, 8), make(6, 8, seed=1), integers(4, 0, 6)
    for call in (lambda: ops.embed(t, w, value), lambda: ops.embed_backward(x, t, 6, value),
                 lambda: ops.linear(x, w, residual=make(4, 6), residual_scale=value),
                 lambda: ops.linear_cross_entropy_grad(x, w, t, grad_scale=value)):
        with pytest.raises(TypeError):
            call()
    # whatever float32 holds is a scale
    assert torch.isinf(ops.embed(t, w, float("inf"))).all()
    assert torch.isfinite(ops.linear(x, w, residual=make(4, 6), residual_scale=torch.tensor(0.5))).all()


@pytest.mark.parametrize("vocab,error", [(-1, ValueError), (0, ValueError), (1 << 31, ValueError), (1 << 40, ValueError),
                                         (1 << 70, ValueError), (6.0, TypeError), ("6", TypeError), (None, TypeError)])
def test_vocabularies(vocab, error):
    """Refused before anything of that size is allocated."""
    x, t = make(4, 8), integers(4, 0, 6)
    with pytest.raises(error):
        ops.embed_backward(x, t, vocab)
