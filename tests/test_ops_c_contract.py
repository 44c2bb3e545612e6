"""What the C entries of the training operators check and report besides
shapes, types and null pointers.  Nothing here reaches a GPU."""
import pytest

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
