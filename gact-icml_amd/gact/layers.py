"""Layers that keep their input in 8 bits and train on it: checkpoints of rows, layer norm and linear layers.

The saved-tensor hooks of the Controller hand the backward pass a whole dequantized tensor.  These operators save their own input as
8-bit codes (a quarter or half of its bytes) and their backward kernels read the codes where they lie: no dequantized copy exists
at any time.  Rounding is to nearest, so a pass is repeatable and needs no seeds.

A checkpoint holds every row in groups of 256 columns, the last of them shorter, with a float scale and minimum each; its codes are those
of ``op_quantize(x.float(), 8, ..., rng_stream="deterministic")`` and, where 256 divides the columns, ``op_dequantize`` takes them.

The public names are in ``gact.ops``; nothing of this is in the reference, whose layers save through the hooks only.
"""
import collections
import math

import torch

from .cpp_extension import _abi

_TYPES = (torch.float32, torch.float16, torch.bfloat16)
_ACTIVATIONS = {None: 0, "gelu": 1, "gelu_tanh": 2, "silu": 3}
MAX_ROWS, MAX_COLS, NORM_MAX_COLS, FEW_ROWS = 0x40000000, 262144, 16384, 64
_GROUP = 256

_stream = torch._C._cuda_getCurrentRawStream

# codes int8 [rows, stride] (stride: the columns rounded up to 16), scale and min float32 [rows, groups]; shape and dtype of the
# tensor it stands for
Checkpoint = collections.namedtuple("Checkpoint", "codes scale min shape dtype")


def _check(t, name, dtype=None, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a tensor" % name)
    if not t.is_cuda:
        raise RuntimeError(name + " must be a CUDA tensor!")
    if t.dtype not in _TYPES or (dtype is not None and t.dtype is not dtype):
        raise RuntimeError("The type of " + name + " is not correct!")
    if device is not None and t.device != device:
        raise RuntimeError(name + " is on another device")


def _rows_of(t, name, most=MAX_COLS):
    """t as [rows, cols] whose columns lie side by side (a view where the strides allow it), rows and cols."""
    if t.dim() < 1:
        raise RuntimeError("The dimension of " + name + " is not correct!")
    cols = t.shape[-1]
    if not 0 < cols <= most:
        raise RuntimeError("%s has %d columns: 1 to %d are taken" % (name, cols, most))
    rows = t.numel() // cols
    if rows > MAX_ROWS:
        raise RuntimeError("%s has more than %d rows" % (name, MAX_ROWS))
    t = _abi.stored(t)
    if t.dim() != 2:
        t = t.reshape(rows, cols)
    if rows and (t.stride(1) != 1 and cols > 1 or (rows > 1 and (t.stride(0) < cols or t.stride(0) > 4 * MAX_COLS))):
        t = t.contiguous()
    return t, rows, cols


def _ld(t):
    """Elements from one row to the next (of a single row: as if it were one of many)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _product_rows(t):
    """t [rows, cols] as the products load it: 16-byte aligned rows of whole 16-byte pieces."""
    piece = 16 // t.element_size()
    rows, cols = t.shape
    if rows <= 1 and cols % piece == 0 and t.data_ptr() % 16 == 0:
        return t, cols
    if rows > 1 and cols % piece == 0 and t.stride(0) % piece == 0 and t.data_ptr() % 16 == 0:
        return t, t.stride(0)
    ld = (cols + 7) // 8 * 8
    out = torch.empty((rows, ld), dtype=t.dtype, device=t.device)
    _call(t, "gact_pad_rows", t.data_ptr(), _abi.dtype_code(t.dtype), rows, cols, _ld(t), out.data_ptr(), ld)
    return out, ld


def _call(t, name, *args):
    _abi.call_on(t.device, getattr(_abi.lib(), name), *args, _stream(t.device.index))


def _workspace(t, size):
    return torch.empty(size, dtype=torch.uint8, device=t.device) if size else None


def _codes_for(rows, cols, like):
    """Room for a checkpoint of [rows, cols]."""
    groups = (cols + _GROUP - 1) // _GROUP
    return (torch.empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=like.device),
            torch.empty((rows, groups), dtype=torch.float32, device=like.device),
            torch.empty((rows, groups), dtype=torch.float32, device=like.device))


def _compress(x):
    rows, cols = x.shape
    codes, scale, mn = _codes_for(rows, cols, x)
    _call(x, "gact_checkpoint", x.data_ptr(), _abi.dtype_code(x.dtype), rows, cols, _ld(x), codes.data_ptr(), codes.stride(0),
          scale.data_ptr(), mn.data_ptr())
    return codes, scale, mn


def _weight_product(grad, codes, scale, mn, cols, dtype):
    """grad [rows, outer] transposed times the checkpoint's values [rows, cols]; grad as _product_rows left it, with its columns."""
    grad, ld, outer = grad
    rows = codes.shape[0]
    if rows == 0:
        return torch.zeros((outer, cols), dtype=dtype, device=codes.device)
    out = torch.empty((outer, cols), dtype=dtype, device=codes.device)
    code = _abi.dtype_code(dtype)
    ws = _workspace(codes, _abi.lib().gact_product_workspace_bytes(code, outer, cols, rows))
    _call(codes, "gact_checkpoint_product", grad.data_ptr(), ld, codes.data_ptr(), codes.stride(0), scale.data_ptr(), mn.data_ptr(), code,
          rows, outer, cols, out.data_ptr(), _abi.ptr(ws))
    return out


# ---- checkpoints ----
def op_checkpoint(input):
    """The 8-bit checkpoint of a float32, float16 or bfloat16 tensor [..., cols]."""
    _check(input, "data")
    x, _, _ = _rows_of(input.detach(), "data")
    return Checkpoint(*_compress(x), input.shape, input.dtype)


def _check_checkpoint(c):
    if not isinstance(c, Checkpoint):
        raise TypeError("a Checkpoint is expected")
    shape = tuple(c.shape)
    cols = shape[-1] if shape else 0
    rows = math.prod(shape[:-1])
    if not 0 < cols <= MAX_COLS or c.dtype not in _TYPES:
        raise RuntimeError("the checkpoint's shape or type is not correct")
    for t, dtype, width in ((c.codes, torch.int8, (cols + 15) // 16 * 16), (c.scale, torch.float32, (cols + 255) // 256),
                            (c.min, torch.float32, (cols + 255) // 256)):
        if not t.is_cuda or t.device != c.codes.device or t.dtype is not dtype or tuple(t.shape) != (rows, width) or not t.is_contiguous() \
                or not _abi.aligned(t):
            raise RuntimeError("the checkpoint's codes, scale or min do not belong to shape %s" % (shape,))
    return rows, cols


def op_restore(checkpoint):
    """The tensor a checkpoint stands for, in its shape and type."""
    rows, cols = _check_checkpoint(checkpoint)
    codes, scale, mn, shape, dtype = checkpoint
    out = torch.empty(tuple(shape), dtype=dtype, device=codes.device)
    _call(codes, "gact_restore", codes.data_ptr(), codes.stride(0), scale.data_ptr(), mn.data_ptr(), _abi.dtype_code(dtype), rows, cols,
          out.data_ptr())
    return out


def op_checkpoint_product(grad, checkpoint):
    """[outer, cols] = grad [..., outer] transposed times the checkpoint's values [..., cols], both as rows: the weight's gradient of a
    linear layer whose input the checkpoint holds.  The values enter the product in the checkpoint's type, as op_restore gives them."""
    rows, cols = _check_checkpoint(checkpoint)
    _check(grad, "grad", checkpoint.dtype, checkpoint.codes.device)
    g, grad_rows, outer = _rows_of(grad.detach(), "grad")
    if grad_rows != rows:
        raise RuntimeError("grad has %d rows, the checkpoint %d" % (grad_rows, rows))
    if rows:
        g, ld = _product_rows(g)
    else:
        ld = outer
    return _weight_product((g, ld, outer), checkpoint.codes, checkpoint.scale, checkpoint.min, cols, checkpoint.dtype)


# ---- layer norm ----
class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, eps, keep):
        x, rows, cols = _rows_of(input, "data", NORM_MAX_COLS)
        y = torch.empty(input.shape, dtype=input.dtype, device=input.device)
        kept = (None, None, None)
        stats = None
        if keep:
            kept = _codes_for(rows, cols, x)
            stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device)
        if rows:
            _call(x, "gact_norm_forward", x.data_ptr(), _ld(x), _abi.ptr(weight), _abi.ptr(bias), _abi.dtype_code(x.dtype), rows, cols, eps,
                  y.data_ptr(), _abi.ptr(kept[0]), kept[0].stride(0) if keep else 0, _abi.ptr(kept[1]), _abi.ptr(kept[2]), _abi.ptr(stats))
        if keep:
            ctx.save_for_backward(weight, stats, *kept)
            ctx.has_bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight, stats, codes, scale, mn = ctx.saved_tensors
        shape, dtype = dy.shape, dy.dtype
        dy, rows, cols = _rows_of(dy, "grad", NORM_MAX_COLS)
        need_w, need_b = weight is not None and ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        make = torch.empty if rows else torch.zeros
        dw = make(cols, dtype=dtype, device=dy.device) if need_w else None
        db = make(cols, dtype=dtype, device=dy.device) if need_b else None
        dx = torch.empty(shape, dtype=dtype, device=dy.device)
        if rows:
            ws = _workspace(dy, _abi.lib().gact_norm_workspace_bytes(rows, cols)) if need_w or need_b else None
            _call(dy, "gact_norm_backward", dy.data_ptr(), _ld(dy), _abi.ptr(weight), codes.data_ptr(), codes.stride(0), scale.data_ptr(),
                  mn.data_ptr(), stats.data_ptr(), _abi.dtype_code(dtype), rows, cols, dx.data_ptr(), _abi.ptr(dw), _abi.ptr(db), _abi.ptr(ws))
        return dx if ctx.needs_input_grad[0] else None, dw, db, None, None


def _vector(t, name, size, like):
    _check(t, name, like.dtype, like.device)
    if tuple(t.shape) != (size,):
        raise RuntimeError("The dimension of " + name + " is not correct!")
    t = _abi.stored(t)
    return t if t.is_contiguous() else t.contiguous()


def _autocast(*tensors, dtype=None):
    """As the torch operator would under autocast: cast, differentiably, to its type there."""
    if not torch.is_autocast_enabled("cuda"):
        return tensors
    dtype = torch.get_autocast_dtype("cuda") if dtype is None else dtype
    return tuple(t.to(dtype) if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _TYPES else t for t in tensors)


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def op_layer_norm(input, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension.  For the backward pass it keeps the 8-bit checkpoint of the input and each row's mean and
    1 / sqrt(var + eps); gradients are those of the checkpoint's values under that mean and deviation."""
    input, weight, bias = _autocast(input, weight, bias, dtype=torch.float32)
    _check(input, "data")
    if input.dim() < 1 or not 0 < input.shape[-1] <= NORM_MAX_COLS:
        raise RuntimeError("layer norm takes 1 to %d columns" % NORM_MAX_COLS)
    cols = input.shape[-1]
    weight = None if weight is None else _vector(weight, "weight", cols, input)
    bias = None if bias is None else _vector(bias, "bias", cols, input)
    return _LayerNorm.apply(input, weight, bias, float(eps), _needs_grad(input, weight, bias))


# ---- linear layers ----
class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, input, weight, bias, residual, activation, needs):
        x, rows, inner = _rows_of(input, "data")
        outer = weight.shape[0]
        code = _abi.dtype_code(x.dtype)
        y = torch.empty(input.shape[:-1] + (outer,), dtype=x.dtype, device=x.device)
        kept, kept_z = (None, None, None), (None, None, None)
        if needs and activation:
            kept_z = _codes_for(rows, outer, x)
        if rows:
            if rows <= FEW_ROWS and kept_z[0] is None:
                a, lda, w, ldw = x, _ld(x), weight, _ld(weight)
            else:
                (a, lda), (w, ldw) = _product_rows(x), _product_rows(weight)
            r = None if residual is None else _rows_of(residual, "residual")[0]
            # whole pieces: behind the last column both are padded copies with zeros there
            piece = 16 // x.element_size()
            depth = inner if a is x and w is weight else (inner + piece - 1) // piece * piece
            _call(x, "gact_linear", a.data_ptr(), lda, w.data_ptr(), ldw, _abi.ptr(bias), _abi.ptr(r), 0 if r is None else _ld(r), activation,
                  code, rows, depth, outer, y.data_ptr(), _abi.ptr(kept_z[0]), 0 if kept_z[0] is None else kept_z[0].stride(0),
                  _abi.ptr(kept_z[1]), _abi.ptr(kept_z[2]))
        if needs:
            if ctx.needs_input_grad[1]:
                kept = _compress(x) if rows else _codes_for(rows, inner, x)
            ctx.save_for_backward(weight, *kept, *kept_z)
            ctx.activation, ctx.has_bias, ctx.inner = activation, bias is not None, inner
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight, codes, scale, mn, z_codes, z_scale, z_mn = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[0], ctx.needs_input_grad[1], ctx.has_bias and ctx.needs_input_grad[2]
        inner, dtype = ctx.inner, dy.dtype
        dresidual = dy if ctx.needs_input_grad[3] else None
        shape = dy.shape[:-1] + (inner,)
        g, rows, outer = _rows_of(dy, "grad")
        if rows == 0:
            zeros = lambda *s: torch.zeros(s, dtype=dtype, device=dy.device)  # noqa: E731
            return (zeros(*shape) if need_x else None, zeros(outer, inner) if need_w else None, zeros(outer) if need_b else None, dresidual,
                    None, None)
        code, L = _abi.dtype_code(dtype), _abi.lib()
        db = torch.empty(outer, dtype=dtype, device=dy.device) if need_b else None
        ld = (outer + 7) // 8 * 8
        piece = 16 // g.element_size()
        fits = rows == 1 and outer % piece == 0 or rows > 1 and outer % piece == 0 and g.stride(0) % piece == 0
        copied = need_x or need_w if ctx.activation else (need_x or need_w) and not (fits and _abi.aligned(g))
        dz = torch.empty((rows, ld), dtype=dtype, device=dy.device) if copied else None
        if copied or need_b:
            ws = _workspace(dy, L.gact_activation_workspace_bytes(rows, outer)) if need_b else None
            _call(dy, "gact_activation_backward", g.data_ptr(), _ld(g), _abi.ptr(z_codes), 0 if z_codes is None else z_codes.stride(0),
                  _abi.ptr(z_scale), _abi.ptr(z_mn), ctx.activation, code, rows, outer, _abi.ptr(dz), ld, _abi.ptr(db), _abi.ptr(ws))
        if dz is None:
            dz, ld = g, _ld(g)
        dx = dw = None
        if need_x:
            w, ldw = _product_rows(weight)
            dx = torch.empty(shape, dtype=dtype, device=dy.device)
            ws = _workspace(dy, L.gact_product_workspace_bytes(code, rows, inner, outer))
            _call(dy, "gact_product", dz.data_ptr(), ld, w.data_ptr(), ldw, code, rows, outer, inner, dx.data_ptr(), _abi.ptr(ws))
        if need_w:
            dw = _weight_product((dz, ld, outer), codes, scale, mn, inner, dtype)
        return dx, dw, db, dresidual, None, None


def op_linear(input, weight, bias=None, activation=None, residual=None):
    """activation(input weight^T + bias) + residual in one kernel; activation None, "gelu", "gelu_tanh" or "silu".

    For the backward pass it keeps the 8-bit checkpoint of the input and, under an activation, of the value it is applied to; the
    gradients are those of the checkpoints' values.  (relu is not among them: its derivative jumps at zero, where 8 bits do not hold
    the sign.)"""
    if activation not in _ACTIVATIONS:
        raise RuntimeError("unknown activation %r (expected one of %s)" % (activation, sorted(k for k in _ACTIVATIONS if k)))
    input, weight, bias, residual = _autocast(input, weight, bias, residual)
    _check(input, "data")
    _check(weight, "weight", input.dtype, input.device)
    if weight.dim() != 2 or input.dim() < 1 or weight.shape[1] != input.shape[-1]:
        raise RuntimeError("weight must be [outer, %s], got %s" % (input.shape[-1] if input.dim() else "-", tuple(weight.shape)))
    outer, inner = weight.shape
    if not (0 < inner <= MAX_COLS and 0 < outer <= MAX_COLS):
        raise RuntimeError("a linear layer takes 1 to %d columns on either side" % MAX_COLS)
    bias = None if bias is None else _vector(bias, "bias", outer, input)
    if residual is not None:
        _check(residual, "residual", input.dtype, input.device)
        if residual.shape != input.shape[:-1] + (outer,):
            raise RuntimeError("residual must have the result's shape %s" % (tuple(input.shape[:-1]) + (outer,),))
    weight = _rows_of(weight, "weight")[0]
    return _Linear.apply(input, weight, bias, residual, _ACTIVATIONS[activation], _needs_grad(input, weight, bias, residual))
