"""The autograd forms do the work that is asked for and no more: none for
gradients where none are recorded, and only the gradients that are wanted."""
import pytest
import torch

import ops_reference as ref
from alphazero_b200 import ops
from test_gpu_ops import integers, laid, make

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


@pytest.mark.parametrize("name", ["none", "relu", "gelu"])
@pytest.mark.parametrize("how", ["plain", "transposed", "offset"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 8), (3, 362, 722), (9, 128, 2050), (16, 96, 4096), (129, 257, 65),
                                   (300, 128, 1024), (4099, 40, 24)])
def test_one_gradient_at_a_time(name, how, m, n, k):
    g, x = make(m, n, seed=4), make(m, k)
    w, z = laid(make(n, k, seed=1, scale=k ** -0.5), how), make(m, n, seed=5)
    want = ref.linear_backward(g, x, w, z, name)
    for wanted in [(True, False, False), (False, True, False), (False, False, True), (True, False, True),
                   (False, True, True), (False, False, False)]:
        got = ops.linear_backward(g, x, w, z, name, bias=wanted[2], input_grad=wanted[0], weight_grad=wanted[1])
        for a, (b, off), asked in zip(got, want, wanted):
            assert (a is not None) == asked
            if asked:
                ref.within(a, b, off)


def test_frozen_inputs_cost_nothing():
    m, n, k = 64, 8192, 4096  # a gradient of w takes 64 MB, everything else under 2
    for frozen in ("w", "x", "wx", "wxb"):
        x, w = make(m, k), make(n, k, seed=1, scale=0.02)
        b, r = make(n, seed=2), make(m, n, seed=3)
        for letter, t in (("x", x), ("w", w), ("b", b), ("r", r)):
            t.requires_grad_(letter not in frozen)
        y = ops.linear_layer(x, w, b, r, "gelu", 0.5)
        g = make(m, n, seed=4)
        inputs = [t for t in (x, w, b, r) if t.requires_grad]
        got, most = peak(lambda: torch.autograd.grad(y, inputs, g, retain_graph=True))
        full = ops.linear_backward(g, x, w, ops.linear(x, w, b, r, "gelu", 0.5, True)[1], "gelu")
        want = [v for t, v in zip((x, w, b, r), (*full, g * 0.5)) if t.requires_grad]
        for a, c in zip(got, want):
            # sums of other splits, each rounded once to 8 bits
            assert (a.double() - c.double()).norm() <= 2.0 ** -8 * c.double().norm()
        assert ("w" in frozen) == (most < n * k * 2)
