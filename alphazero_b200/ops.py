"""Training operators of a move-sequence policy over torch CUDA tensors:
embedding lookup, linear layer and linear cross entropy, each with its
gradient, over the C ABI of include/minigo_ops.h (libminigo_cuda.so).

Every function enqueues its kernels on the current stream of the tensors'
device and returns without waiting, like torch's own; scratch comes from
torch's allocator.  Inputs are read where they lie, with any strides; outputs
are new dense tensors of the inputs' type.  Arguments that do not fit raise
ValueError (wrong shapes or values) or TypeError (wrong types or devices);
failures of the library raise RuntimeError.  There is no CPU fallback.

``embedding``, ``linear_layer`` and ``cross_entropy_loss`` are the same
operators for torch's autograd (first derivatives; a second one raises).  The
others record nothing: what they return requires no gradient, whatever their
inputs do.  The reference trains with torch on its own (scripts/train.py) and
has no counterpart.
"""
from __future__ import annotations

import ctypes
import struct
from operator import index

import torch
from torch.autograd.function import once_differentiable

from . import engine

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_FLOAT_LIMIT = 2.0 ** 128  # a float32 is below it
_INDEX_BYTES = {torch.int64: 8, torch.int32: 4}

# The argument structs of minigo_ops.h, field by field.
_EMBED = struct.Struct("3P5qf3i")
_EMBED_BACKWARD = struct.Struct("3P5qf3i")
_LINEAR = struct.Struct("6P9qf3i")
_LINEAR_BACKWARD = struct.Struct("7P11q4i")
_CROSS_ENTROPY = struct.Struct("9P8qf3i")

_LIB = None


def lib() -> ctypes.CDLL:
    """libminigo_cuda.so with the operators' signatures."""
    global _LIB
    if _LIB is None:
        L = engine.lib()
        vp = ctypes.c_void_p
        size = ctypes.POINTER(ctypes.c_size_t)
        L.mg_op_error.restype = ctypes.c_char_p
        L.mg_op_error.argtypes = []
        L.mg_op_synchronize.argtypes = [ctypes.c_int, vp]
        L.mg_embed.argtypes = [vp, vp]
        for name in ("mg_embed_backward", "mg_linear", "mg_linear_backward", "mg_cross_entropy"):
            getattr(L, name).argtypes = [vp, vp, ctypes.c_size_t, vp]
            getattr(L, name + "_workspace").argtypes = [vp, size]
        _LIB = L
    return _LIB


def _raise(code: int):
    message = lib().mg_op_error().decode() or f"error {code}"
    raise ValueError(message) if code == -1 else RuntimeError(message)


# The current stream of a device by index, without a Stream object (a torch without CUDA has none).
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _pack(layout: struct.Struct, *values) -> bytes:
    try:
        return layout.pack(*values)
    except struct.error as e:  # everything else has been checked
        raise TypeError("a scale must be a number") from e


def _call(name: str, args: bytes, like, device: int) -> None:
    L = _LIB or lib()
    need = ctypes.c_size_t()
    code = getattr(L, name + "_workspace")(args, ctypes.byref(need))
    if code:
        _raise(code)
    size = need.value
    # torch's allocator orders the block's reuse after this stream's work
    w = like.new_empty(size, dtype=torch.uint8) if size else None
    code = getattr(L, name)(args, w.data_ptr() if size else None, size, _stream(device))
    if code:
        _raise(code)


def synchronize(device=None) -> None:
    """Waits for the current stream; raises RuntimeError if a kernel of these
    operators gave up a bounded wait (its outputs are then invalid)."""
    d = torch.device("cuda" if device is None else device)
    index = d.index if d.index is not None else torch.cuda.current_device()
    code = lib().mg_op_synchronize(index, _stream(index))
    if code:
        _raise(code)


# ---- argument checks ----

def _on_gpu(t, name: str) -> int:
    """The index of the tensor's device."""
    if isinstance(t, torch.Tensor) and t.is_cuda:
        return t.get_device()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, not {type(t).__name__}")
    raise TypeError(f"{name} must be a CUDA tensor (it is on {t.device})")


def _same(t, name: str, like, what: str, device: int) -> None:
    if _on_gpu(t, name) != device:
        raise TypeError(f"{name} is on {t.device}, {what} on {like.device}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} is {t.dtype}, {what} {like.dtype}")


def _dtype(t, name: str, wide: bool) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None or (code == 2 and not wide):
        raise TypeError(f"{name} must be bfloat16{', float16 or float32' if wide else ' or float16'}, "
                        f"not {t.dtype}")
    return code


def _indices(t, name: str, like, device: int) -> int:
    if _on_gpu(t, name) != device:
        raise TypeError(f"{name} is on {t.device}, expected {like.device}")
    b = _INDEX_BYTES.get(t.dtype)
    if b is None:
        raise TypeError(f"{name} must be int64 or int32, not {t.dtype}")
    return b


def _flat(t):
    """t as a vector, and its stride."""
    v = t if t.dim() == 1 else t.reshape(-1)
    return v, v.stride()[0]


def _matrix(t, name: str, cols=None):
    """t [..., cols] as [rows, cols]; a copy only where the leading
    dimensions cannot be one."""
    shape = t.shape
    if not shape:
        raise ValueError(f"{name} must have at least one dimension")
    if cols is not None and shape[-1] != cols:
        raise ValueError(f"{name} has {shape[-1]} columns, expected {cols}")
    if len(shape) == 2:
        return t
    if shape[-1] == 0:
        raise ValueError(f"{name} has no columns")
    return t.reshape(-1, shape[-1])


def _weight(t, name: str, like, what: str, device: int) -> None:
    _same(t, name, like, what, device)
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix, not {tuple(t.shape)}")


def _vector(t, name: str, n: int, like, what: str, device: int):
    _same(t, name, like, what, device)
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must have shape ({n},), not {tuple(t.shape)}")
    return t.contiguous()


def _rows(t):
    """t with unit column stride."""
    return t if t.stride()[1] == 1 or t.shape[1] == 1 else t.contiguous()


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _activation(name: str) -> int:
    code = ACTIVATIONS.get(name)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, not {name!r}")
    return code


# ---- embedding ----

def embed(tokens, table, scale: float = 1.0):
    """``scale * table[tokens]``: tokens [...] int64 or int32, table
    [vocab, dim] bfloat16, float16 or float32 -> [..., dim].  A token outside
    [0, vocab) is padding and gives a zero row."""
    d = _on_gpu(table, "table")
    dt = _dtype(table, "table", True)
    tb = _indices(tokens, "tokens", table, d)
    if table.dim() != 2:
        raise ValueError(f"table must be a matrix, not {tuple(table.shape)}")
    vocab, dim = table.shape
    t, t_stride = _flat(tokens)
    row, column = table.stride()
    if column != 1 and dim != 1:
        table = table.contiguous()
        row = dim
    n = t.numel()
    out = table.new_empty((n, dim) if t is tokens else (*tokens.shape, dim))
    code = (_LIB or lib()).mg_embed(_pack(_EMBED, t.data_ptr(), table.data_ptr(), out.data_ptr(), n, vocab,
                                                 dim, t_stride, row, scale, dt, tb, d), _stream(d))
    if code:
        _raise(code)
    return out


def embed_backward(grad, tokens, vocab: int, scale: float = 1.0):
    """Gradient of ``embed`` with respect to its table: [vocab, dim], the
    rows of grad [..., dim] summed by token in 32 bits, times scale."""
    d = _on_gpu(grad, "grad")
    dt = _dtype(grad, "grad", True)
    tb = _indices(tokens, "tokens", grad, d)
    if grad.shape[:-1] != tokens.shape:
        raise ValueError(f"grad {tuple(grad.shape)} does not match tokens {tuple(tokens.shape)}")
    g = _rows(_matrix(grad, "grad"))
    t, t_stride = _flat(tokens)
    n, dim = g.shape
    vocab = index(vocab)
    if not 0 < vocab < 1 << 31:
        raise ValueError(f"vocab must be from 1 to 2^31 - 1, not {vocab}")
    out = grad.new_empty((vocab, dim))
    _call("mg_embed_backward",
          _pack(_EMBED_BACKWARD, t.data_ptr(), g.data_ptr(), out.data_ptr(), n, vocab, dim, t_stride,
                g.stride(0), scale, dt, tb, d), grad, d)
    return out


# ---- linear layer ----

def linear(x, weight, bias=None, residual=None, activation: str = "none",
           residual_scale: float = 1.0, keep_preactivation: bool = False):
    """``act(x @ weight.T + bias) + residual_scale * residual`` in one pass:
    x [..., k], weight [n, k], bias [n], residual [..., n] -> [..., n], in
    bfloat16 or float16 with 32-bit sums.  activation is "none", "relu",
    "silu" or "gelu" (the erf form).  With keep_preactivation returns
    (y, z), z = x @ weight.T + bias being what ``linear_backward`` needs."""
    d = _on_gpu(x, "x")
    dt = _dtype(x, "x", False)
    act = _activation(activation)
    _weight(weight, "weight", x, "x", d)
    n, k = weight.shape
    x2 = _matrix(x, "x", k)
    b = None if bias is None else _vector(bias, "bias", n, x, "x", d)
    shape = (x2.shape[0], n) if x2 is x else (*x.shape[:-1], n)
    r, r_row, r_col = None, 0, 0
    if residual is not None:
        _same(residual, "residual", x, "x", d)
        if residual.shape != shape:
            raise ValueError(f"residual must have shape {tuple(shape)}, not {tuple(residual.shape)}")
        r = _matrix(residual, "residual")
        r_row, r_col = r.stride()
    y = x.new_empty(shape)
    z = x.new_empty(shape) if keep_preactivation else None
    _call("mg_linear",
          _pack(_LINEAR, x2.data_ptr(), weight.data_ptr(), _ptr(b), _ptr(r), y.data_ptr(), _ptr(z),
                x2.shape[0], n, k, *x2.stride(), *weight.stride(), r_row, r_col, residual_scale,
                act, dt, d), x, d)
    return (y, z) if keep_preactivation else y


def linear_backward(grad, x, weight, preactivation=None, activation: str = "none", bias: bool = True,
                    input_grad: bool = True, weight_grad: bool = True):
    """Gradients (dx, dw, db) of ``linear`` from grad = dL/dy [..., n] and
    the z that it kept (needed unless activation is "none"); dx is None, and
    not computed, with input_grad=False, dw with weight_grad=False, db with
    bias=False.  The residual's gradient is residual_scale * grad."""
    d = _on_gpu(grad, "grad")
    dt = _dtype(grad, "grad", False)
    act = _activation(activation)
    _same(x, "x", grad, "grad", d)
    _weight(weight, "weight", grad, "grad", d)
    n, k = weight.shape
    g, x2 = _matrix(grad, "grad", n), _matrix(x, "x", k)
    if grad.shape[:-1] != x.shape[:-1]:
        raise ValueError(f"grad {tuple(grad.shape)} does not match x {tuple(x.shape)}")
    z, z_row, z_col = None, 0, 0
    if act:
        if preactivation is None:
            raise ValueError(f"the backward pass of {activation!r} needs the preactivation")
        _same(preactivation, "preactivation", grad, "grad", d)
        if preactivation.shape != grad.shape:
            raise ValueError(f"preactivation must have shape {tuple(grad.shape)}, not "
                             f"{tuple(preactivation.shape)}")
        z = _matrix(preactivation, "preactivation")
        z_row, z_col = z.stride()
    dx = x.new_empty(x.shape) if input_grad else None
    dw = x.new_empty((n, k)) if weight_grad else None
    db = x.new_empty((n,)) if bias else None
    _call("mg_linear_backward",
          _pack(_LINEAR_BACKWARD, g.data_ptr(), x2.data_ptr(), weight.data_ptr(), _ptr(z),
                _ptr(dx), _ptr(dw), _ptr(db), g.shape[0], n, k, *g.stride(), *x2.stride(),
                *weight.stride(), z_row, z_col, act, dt, d, 0), x, d)
    return dx, dw, db


# ---- linear cross entropy ----

def _cross_entropy(x, weight, targets, bias, grad_scale, gradients):
    d = _on_gpu(x, "x")
    dt = _dtype(x, "x", False)
    _weight(weight, "weight", x, "x", d)
    vocab, dim = weight.shape
    x2 = _matrix(x, "x", dim)
    tb = _indices(targets, "targets", x, d)
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"targets {tuple(targets.shape)} do not match x {tuple(x.shape)}")
    t, t_stride = _flat(targets)
    b = None if bias is None else _vector(bias, "bias", vocab, x, "x", d)
    loss = x.new_empty((), dtype=torch.float32)
    rows = x.new_empty(targets.shape, dtype=torch.float32)
    dx = dw = db = None
    if gradients:
        dx = x.new_empty(x.shape)
        dw = x.new_empty((vocab, dim))
        db = x.new_empty((vocab,)) if b is not None else None
    _call("mg_cross_entropy",
          _pack(_CROSS_ENTROPY, x2.data_ptr(), weight.data_ptr(), _ptr(b), t.data_ptr(),
                loss.data_ptr(), rows.data_ptr(), _ptr(dx), _ptr(dw), _ptr(db), t.shape[0], vocab,
                dim, *x2.stride(), *weight.stride(), t_stride, grad_scale, dt, tb, d), x, d)
    return loss, rows, dx, dw, db


def linear_cross_entropy(x, weight, targets, bias=None):
    """(loss, row_loss) of softmax(x @ weight.T + bias) against target
    indices, without keeping the logits: x [..., dim], weight [vocab, dim],
    bias [vocab] (-inf bans an entry), targets [...] int64 or int32; the
    losses are float32.  A target outside [0, vocab) leaves its row out
    (row_loss 0); loss is the mean over the other rows, 0 if there is none."""
    return _cross_entropy(x, weight, targets, bias, 1.0, False)[:2]


def linear_cross_entropy_grad(x, weight, targets, bias=None, grad_scale: float = 1.0):
    """(loss, row_loss, dx, dw, db): ``linear_cross_entropy`` and the
    gradients of grad_scale * loss (db None without a bias) in one call.
    float16 gradients need a grad_scale that keeps them in range."""
    return _cross_entropy(x, weight, targets, bias, grad_scale, True)


# ---- autograd ----

def _recorded(*inputs) -> bool:
    """Whether a gradient can be asked for.  (Inside a Function's forward
    this is not to be known: gradients are off there in any case, and
    needs_input_grad tells what inputs require, under no_grad as well.)"""
    return torch.is_grad_enabled() and any(getattr(t, "requires_grad", False) for t in inputs)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, scale):
        ctx.save_for_backward(tokens)
        ctx.vocab, ctx.scale = table.shape[0], scale
        return embed(tokens, table, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        (tokens,) = ctx.saved_tensors
        return None, embed_backward(grad, tokens, ctx.vocab, ctx.scale), None


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, residual_scale):
        keep = activation != "none" and any(ctx.needs_input_grad[:3])
        out = linear(x, weight, bias, residual, activation, residual_scale, keep)
        y, z = out if keep else (out, None)
        ctx.save_for_backward(x, weight, z)
        ctx.activation, ctx.residual_scale = activation, residual_scale
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, z = ctx.saved_tensors
        x_grad, w_grad, b_grad, r_grad = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if x_grad or w_grad or b_grad:
            dx, dw, db = linear_backward(grad, x, weight, z, ctx.activation, b_grad, x_grad, w_grad)
        dr = grad * ctx.residual_scale if r_grad else None
        return dx, dw, db, dr, None, None


class _CrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, targets, grad_scale):
        loss, _, dx, dw, db = linear_cross_entropy_grad(x, weight, targets, bias, grad_scale)
        ctx.save_for_backward(dx, dw, db)
        ctx.grad_scale = grad_scale
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        factor = grad / ctx.grad_scale
        dx, dw, db = ((t * factor).to(t.dtype) if wanted else None
                      for t, wanted in zip(ctx.saved_tensors, ctx.needs_input_grad))
        return dx, dw, db, None, None


def embedding(tokens, table, scale: float = 1.0):
    """``embed`` for autograd."""
    if not _recorded(table):
        return embed(tokens, table, float(scale))
    return _Embedding.apply(tokens, table, float(scale))


def linear_layer(x, weight, bias=None, residual=None, activation: str = "none",
                 residual_scale: float = 1.0):
    """``linear`` for autograd."""
    if not _recorded(x, weight, bias, residual):
        return linear(x, weight, bias, residual, activation, float(residual_scale))
    return _Linear.apply(x, weight, bias, residual, activation, float(residual_scale))


def cross_entropy_loss(x, weight, targets, bias=None, grad_scale: float = 1.0):
    """The loss of ``linear_cross_entropy`` for autograd.  The gradients are
    made with the loss, of grad_scale * loss, and multiplied by the incoming
    gradient / grad_scale when the backward pass reaches them; where none can
    be asked for, only the loss is.  So grad_scale is a finite number that is
    not 0, in the range of float32."""
    if not 0.0 < abs(float(grad_scale)) < _FLOAT_LIMIT:
        raise ValueError(f"grad_scale must be finite and not 0, not {grad_scale}")
    if not _recorded(x, weight, bias):
        return linear_cross_entropy(x, weight, targets, bias)[0]
    return _CrossEntropy.apply(x, weight, bias, targets, float(grad_scale))
