"""What the training operators refuse, at the C entries and in Python.
Nothing here reaches a GPU: arguments are checked before any CUDA call."""
import ctypes
import os
import re

import pytest
import torch

from alphazero_b200 import build, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def L():
    build.build_cuda()
    return ops.lib()


def test_library_exports_the_operators(L):
    text = open(os.path.join(ROOT, "include", "minigo_ops.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(mg_[a-z0-9_]+)\s*\(", text)))
    assert len(names) >= 11
    for n in names:
        getattr(L, n)


def linear_args(**k):
    v = dict(x=256, w=256, b=0, r=0, y=256, z=0, m=4, n=8, k=8, x_row=8, x_col=1, w_row=8, w_col=1,
             r_row=0, r_col=0, scale=1.0, act=0, dt=0, dev=0)
    v.update(k)
    return ops._LINEAR.pack(*v.values())


def embed_args(**k):
    v = dict(tokens=256, table=256, out=256, n=4, vocab=8, dim=8, ts=1, row=8, scale=1.0, dt=0, tb=8, dev=0)
    v.update(k)
    return ops._EMBED.pack(*v.values())


def backward_args(**k):
    v = dict(g=256, x=256, w=256, z=256, dx=256, dw=256, db=0, m=4, n=8, k=8, gr=8, gc=1, xr=8, xc=1,
             wr=8, wc=1, zr=8, zc=1, act=1, dt=0, dev=0, reserved=0)
    v.update(k)
    return ops._LINEAR_BACKWARD.pack(*v.values())


def entropy_args(**k):
    v = dict(x=256, w=256, b=0, t=256, loss=256, rows=256, dx=0, dw=0, db=0, n=4, vocab=8, dim=8,
             xr=8, xc=1, wr=8, wc=1, ts=1, scale=1.0, dt=0, tb=8, dev=0)
    v.update(k)
    return ops._CROSS_ENTROPY.pack(*v.values())


def refused(L, name, args, word):
    need = ctypes.c_size_t(77)
    calls = [lambda: getattr(L, name + "_workspace")(args, ctypes.byref(need)),
             lambda: getattr(L, name)(args, None, 0, None)]
    if name == "mg_embed":
        calls = [lambda: L.mg_embed(args, None)]
    for call in calls:
        assert call() == -1
        assert word in L.mg_op_error().decode()
    assert need.value == 77


@pytest.mark.parametrize("change,word", [
    (dict(n=0), "n >= 1"), (dict(k=0), "k >= 1"), (dict(m=-1), "m >= 0"), (dict(m=1 << 31), "2^31"),
    (dict(dt=2), "dtype"), (dict(dt=7), "dtype"), (dict(act=4), "MG_ACT"), (dict(act=-1), "MG_ACT"),
    (dict(x=0), "null"), (dict(w=0), "null"), (dict(y=0), "null"), (dict(x_row=-8), "negative"),
    (dict(w_col=-1), "negative"), (dict(r=256, r_row=-1), "negative"),
])
def test_linear(L, change, word):
    refused(L, "mg_linear", linear_args(**change), word)


@pytest.mark.parametrize("change,word", [
    (dict(n=0), "n >= 1"), (dict(k=0), "k >= 1"), (dict(dt=2), "dtype"), (dict(act=9), "MG_ACT"),
    (dict(g=0), "grad"), (dict(w=0), "weight"), (dict(x=0), "x"), (dict(z=0), "needs z"),
    (dict(zr=-1), "negative"), (dict(gc=-1), "negative"),
])
def test_linear_backward(L, change, word):
    refused(L, "mg_linear_backward", backward_args(**change), word)


@pytest.mark.parametrize("change,word", [
    (dict(vocab=0), "vocab >= 1"), (dict(dim=0), "dim >= 1"), (dict(n=-1), "n >= 0"), (dict(tb=2), "int32"),
    (dict(dt=3), "dtype"), (dict(tokens=0), "null"), (dict(table=0), "null"), (dict(out=0), "null"),
    (dict(vocab=1 << 31), "2^31"), (dict(ts=-1), "negative"), (dict(row=-8), "negative"),
])
def test_embed(L, change, word):
    refused(L, "mg_embed", embed_args(**change), word)
    refused(L, "mg_embed_backward", embed_args(**change), word)  # the same layout of fields


@pytest.mark.parametrize("change,word", [
    (dict(vocab=0), "vocab >= 1"), (dict(dim=0), "dim >= 1"), (dict(n=-1), "n >= 0"), (dict(dt=2), "dtype"),
    (dict(tb=1), "int32"), (dict(w=0), "null"), (dict(loss=0), "null"), (dict(t=0), "null"),
    (dict(rows=0), "null"), (dict(dx=256), "both dx and dw"), (dict(dw=256), "both dx and dw"),
    (dict(db=256), "both dx and dw"), (dict(dx=256, dw=256, db=256), "db goes with a bias"),
    (dict(dx=256, dw=256, b=256), "db goes with a bias"), (dict(ts=-1), "negative"),
    (dict(xr=-1), "negative"),
])
def test_cross_entropy(L, change, word):
    refused(L, "mg_cross_entropy", entropy_args(**change), word)


def test_null_arguments(L):
    need = ctypes.c_size_t()
    assert L.mg_embed(None, None) == -1
    for name in ("mg_embed_backward", "mg_linear", "mg_linear_backward", "mg_cross_entropy"):
        assert getattr(L, name)(None, None, 0, None) == -1
        assert getattr(L, name + "_workspace")(None, ctypes.byref(need)) == -1
    assert L.mg_linear_workspace(linear_args(), None) == -1


def test_workspace_sizes_need_no_gpu(L):
    need = ctypes.c_size_t()
    for name, args in (("mg_embed_backward", embed_args()), ("mg_linear", linear_args()),
                       ("mg_linear_backward", backward_args()), ("mg_cross_entropy", entropy_args()),
                       ("mg_cross_entropy", entropy_args(dx=256, dw=256))):
        assert getattr(L, name + "_workspace")(args, ctypes.byref(need)) == 0
    # the piece of the logits is bounded, however many rows there are
    big, sizes = 1 << 17, []
    for n in (1 << 16, 1 << 20):
        a = entropy_args(n=n, vocab=big, dx=256, dw=256)
        assert L.mg_cross_entropy_workspace(a, ctypes.byref(need)) == 0
        sizes.append(need.value)
    assert sizes[1] - sizes[0] < 64 * (1 << 20) and sizes[1] < 4 << 30


def test_python_refuses_cpu_tensors_and_other_objects():
    f = torch.zeros(4, 8, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.embed(t, f), lambda: ops.embed_backward(f, t, 9), lambda: ops.linear(f, f),
                 lambda: ops.linear_backward(f, f, f), lambda: ops.linear_cross_entropy(f, f, t),
                 lambda: ops.linear_cross_entropy_grad(f, f, t)):
        with pytest.raises(TypeError, match="CUDA tensor"):
            call()
    with pytest.raises(TypeError, match="torch tensor"):
        ops.linear([1.0], f)


@pytest.mark.gpu
def test_python_refuses_wrong_tensors():
    def f(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    x, w = f(4, 8), f(6, 8)
    for error, call in (
            (TypeError, lambda: ops.linear(f(4, 8, dtype=torch.float32), f(6, 8, dtype=torch.float32))),
            (TypeError, lambda: ops.linear(x, f(6, 8, dtype=torch.float16))),
            (TypeError, lambda: ops.linear(x, w.cpu())),
            (ValueError, lambda: ops.linear(x, f(6, 7))),
            (ValueError, lambda: ops.linear(x, w, bias=f(5))),
            (ValueError, lambda: ops.linear(x, w, residual=f(4, 5))),
            (ValueError, lambda: ops.linear(x, w, activation="tanh")),
            (ValueError, lambda: ops.linear(x, f(0, 8))),
            (ValueError, lambda: ops.linear_backward(f(4, 6), x, w, activation="relu")),
            (ValueError, lambda: ops.linear_backward(f(3, 6), x, w)),
            (ValueError, lambda: ops.linear_backward(f(4, 6), x, w, f(4, 5), "relu")),
            (TypeError, lambda: ops.embed(t.float(), w)),
            (TypeError, lambda: ops.embed(t, w.double())),
            (ValueError, lambda: ops.embed(t, f(6))),
            (ValueError, lambda: ops.embed_backward(f(5, 8), t, 6)),
            (ValueError, lambda: ops.embed_backward(x, t, 0)),
            (ValueError, lambda: ops.linear_cross_entropy(x, w, t[:3])),
            (TypeError, lambda: ops.linear_cross_entropy(x, w, t.to(torch.int16))),
            (ValueError, lambda: ops.linear_cross_entropy_grad(x, w, t, bias=f(5)))):
        with pytest.raises(error):
            call()
