"""What the C entries of the training operators check and report besides
shapes, types and null pointers.  Nothing here reaches a GPU."""
import ctypes

import pytest
import torch

from alphazero_b200 import build, ops
from test_ops_refusals import backward_args, embed_args, entropy_args, linear_args, refused


@pytest.fixture(scope="module")
def L():
    build.build_cuda()
    return ops.lib()


@pytest.mark.parametrize("name,args,words", [
    ("mg_linear", linear_args, dict(x="x", w="weight", b="bias", r="residual", y="y", z="z")),
    ("mg_linear_backward", backward_args, dict(g="grad", x="x", w="weight", z="z", dx="dx", dw="dw", db="db")),
    ("mg_cross_entropy", lambda **k: entropy_args(**{**dict(b=256, dx=256, dw=256, db=256), **k}),
     dict(x="x", w="weight", b="bias", t="targets", loss="loss", rows="row_loss", dx="dx", dw="dw", db="db")),
    ("mg_embed", lambda **k: embed_args(dt=2, **k), dict(tokens="tokens", table="table", out="out")),
    ("mg_embed_backward", lambda **k: embed_args(dt=2, **k), dict(tokens="tokens", table="grad", out="d_table")),
])
def test_pointers_inside_an_element_are_refused(L, name, args, words):
    for field, word in words.items():
        refused(L, name, args(**{field: 257}), word + " is not aligned")
    wide = {"t": "targets", "tokens": "tokens", "loss": "loss", "rows": "row_loss"}
    if name.startswith("mg_embed"):
        wide.update({k: v for k, v in words.items() if k != "tokens"})
    for field, word in wide.items():
        if field in words:  # 2 bytes past an element of 4 or 8
            refused(L, name, args(**{field: 258}), word + " is not aligned")


@pytest.mark.parametrize("vocab", [510, 131072, 1000003])
@pytest.mark.parametrize("bias", [False, True])
def test_gradient_scratch_does_not_grow_with_the_rows(L, vocab, bias):
    """Rows are taken in pieces; what is kept between pieces has the size of
    a gradient, and of a loss per 128 rows."""
    need, sizes = ctypes.c_size_t(), []
    rows = (1 << 16, 1 << 20) if vocab > 510 else (3 << 20, 24 << 20)
    for n in rows:
        a = entropy_args(n=n, vocab=vocab, dx=256, dw=256, b=256 * bias, db=256 * bias)
        assert L.mg_cross_entropy_workspace(a, ctypes.byref(need)) == 0
        sizes.append(need.value)
    assert sizes[1] - sizes[0] < 64 << 20 and sizes[1] < 2 << 30


@pytest.mark.parametrize("vocab", [82, 510, 700, 65536, 1000003])
def test_scoring_scratch_does_not_grow_with_the_rows(L, vocab):
    """Without gradients too: statistics per row and block of columns are kept for
    a piece of the rows."""
    need, sizes = ctypes.c_size_t(), []
    rows = (1 << 18, 1 << 22) if vocab > 700 else (1 << 27, 1 << 29)
    for n in rows:
        assert L.mg_cross_entropy_workspace(entropy_args(n=n, vocab=vocab), ctypes.byref(need)) == 0
        sizes.append(need.value)
    assert sizes[1] - sizes[0] < 64 << 20 and sizes[1] < 2 << 30


@pytest.mark.parametrize("scale", [0.0, -0.0, float("inf"), float("nan"), 1e39])
def test_a_gradient_scale_that_cannot_be_divided_by_is_refused(scale):
    f, t = torch.zeros(4, 8, dtype=torch.bfloat16, requires_grad=True), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(ValueError, match="grad_scale"):
        ops.cross_entropy_loss(f, f, t, grad_scale=scale)
