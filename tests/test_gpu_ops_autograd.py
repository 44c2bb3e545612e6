"""The autograd forms do the work that is asked for and no more: none for
gradients where none are recorded, and only the gradients that are wanted."""
import pytest
import torch

from alphazero_b200 import ops
from test_gpu_ops import integers, make

pytestmark = pytest.mark.gpu


def peak(call):
    """(result, bytes allocated at most during the call beyond those before)."""
    call()  # the kernels are there
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = call()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_no_gradient_work_where_none_is_recorded(mode):
    n, vocab, dim = 512, 60000, 256
    x, w = make(n, dim).requires_grad_(), make(vocab, dim, seed=1, scale=0.1).requires_grad_()
    b, t = make(vocab, seed=2).requires_grad_(), integers(n, 0, vocab)
    want = ops.linear_cross_entropy(x, w, t, b)[0]
    with mode():
        loss, most = peak(lambda: ops.cross_entropy_loss(x, w, t, b))
    assert torch.equal(loss, want) and not loss.requires_grad
    assert most < vocab * dim * 2  # a gradient of w alone takes as much

    m = 8192
    x = make(m, dim).requires_grad_()
    w, r = make(1024, dim, seed=1, scale=0.1).requires_grad_(), make(m, 1024, seed=2).requires_grad_()
    with mode():
        y, most = peak(lambda: ops.linear_layer(x, w, None, r, "gelu"))
    assert torch.equal(y, ops.linear(x, w, None, r, "gelu")) and not y.requires_grad
    assert most < 2 * m * 1024 * 2  # y alone, no z

    with mode():
        e = ops.embedding(t, w[:100], 2.0)
    assert torch.equal(e, ops.embed(t, w[:100], 2.0)) and not e.requires_grad


def test_nothing_is_recorded_for_inputs_without_gradients():
    x, w, t = make(40, 64), make(200, 64, seed=1), integers(40, 0, 200)
    loss = ops.cross_entropy_loss(x, w, t)
    y = ops.linear_layer(x, w, activation="silu")
    assert not loss.requires_grad and not y.requires_grad
    assert torch.equal(loss, ops.linear_cross_entropy(x, w, t)[0])
    assert torch.equal(y, ops.linear(x, w, activation="silu"))


def test_wrong_arguments_are_refused_by_the_autograd_forms_too():
    x, w = make(4, 8), make(6, 8, seed=1)
    for grad in (False, True):
        w.requires_grad_(grad)
        with pytest.raises(ValueError):
            ops.linear_layer(x, w, activation="tanh")
        with pytest.raises(TypeError):
            ops.linear_layer([1.0], w)
        with pytest.raises(TypeError):
            ops.embedding(torch.zeros(3, device="cuda"), w)
        with pytest.raises(ValueError):
            ops.cross_entropy_loss(x, w, integers(3, 0, 6))
