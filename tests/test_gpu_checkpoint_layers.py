"""Checkpoints of rows, layer norm and linear layers on the GPU against their formulas in 64 bits.  The bounds are those of 32-bit
sums over the given lengths and of one rounding to the result's type each, worked out element by element from the inputs."""
import itertools

import pytest
import torch

from gact import ops
from gact.cpp_extension import _abi
from layer_reference import FUNCTION, MAX_SLOPE, U, activation, close, codes_of, gamma, half_step, least, spread, values_of

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# ---- checkpoints ----
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (2, 255), (5, 256), (4, 257), (33, 264), (17, 512), (9, 771), (70, 1000), (3, 4096), (37, 121), (300, 128), (41, 129)])
def test_checkpoint_codes_and_values(rows, cols, dtype):
    x = normal(rows, cols, dtype=dtype)
    kept = ops.op_checkpoint(x)
    codes, scale, mn = codes_of(x)
    assert torch.equal(kept.codes.view(torch.uint8)[:, :cols], codes)
    assert torch.equal(kept.scale, scale) and torch.equal(kept.min, mn)
    back = ops.op_restore(kept)
    assert back.shape == x.shape and back.dtype is dtype
    want, off = values_of(kept.codes, kept.scale, kept.min, cols)
    close(back, want, off + half_step(dtype) * want.abs() + least(dtype), "values")
    # a code is at most half a step of its group off x: |v - x| <= step / 2 (with float32's own roundings), and the value v, which is at
    # most |x| + step / 2, is rounded to the type: |T(v) - x| <= step / 2 + h (|x| + step / 2)
    step = 1.0002 / spread(kept.scale, cols).double()
    close(back, x.double(), step / 2 + off + half_step(dtype) * (x.double().abs() + step / 2) + 4e-6 / 255, "input")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_checkpoint_is_the_packages_format_where_groups_fill_rows(dtype):
    x = normal(37, 1024, dtype=dtype)
    kept = ops.op_checkpoint(x)
    q, bits, scale, mn = ops.op_quantize(x.float(), 8, 0, rng_stream="deterministic")
    assert torch.equal(kept.codes.view(-1), q[:kept.codes.numel()])
    assert torch.equal(kept.scale.view(-1), scale.view(-1)) and torch.equal(kept.min.view(-1), mn.view(-1))
    back = ops.op_dequantize([kept.codes.view(-1), 8, kept.scale.view(-1, 1, 1), kept.min.view(-1, 1, 1)], x.shape)
    want, off = values_of(kept.codes, kept.scale, kept.min, 1024)
    close(back, want, off, "op_dequantize")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_checkpoint_of_awkward_rows(dtype):
    """Constant groups, huge ranges, a single value in the last group."""
    x = torch.zeros(6, 257, dtype=torch.float32)
    x[1] = 1.5
    x[2, 3] = 60000.0
    x[3, 5] = -60000.0
    x[4, 256] = 7.0
    x[5] = torch.linspace(-1e-3, 1e-3, 257)
    x = x.to(dtype).cuda()
    kept = ops.op_checkpoint(x)
    codes, scale, mn = codes_of(x)
    assert torch.equal(kept.codes.view(torch.uint8)[:, :257], codes) and torch.equal(kept.scale, scale) and torch.equal(kept.min, mn)
    back = ops.op_restore(kept)
    assert torch.equal(back[0], x[0]) and torch.equal(back[1], x[1]) and back[4, 256] == 7.0


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_checkpoint_takes_strides_views_and_more_dimensions(dtype):
    base = normal(40, 600, dtype=dtype)
    views = [base[:, 3:300], base[::2], base[:, ::2], base.t(), base[:1].expand(5, 600), base.view(2, 4, 5, 600)[:, :, 1], base[7]]
    for v in views:
        kept = ops.op_checkpoint(v)
        plain = ops.op_checkpoint(v.contiguous().clone())
        cols = v.shape[-1]
        assert torch.equal(kept.codes[:, :cols], plain.codes[:, :cols]) and torch.equal(kept.scale, plain.scale)
        assert ops.op_restore(kept).shape == v.shape


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,outer,cols", [(1, 1, 1), (1, 8, 256), (5, 3, 9), (64, 128, 128), (65, 130, 257), (200, 64, 771), (1000, 129, 384),
                                             (2100, 300, 520), (700, 1030, 264)])
def test_checkpoint_product(rows, outer, cols, dtype):
    x, g = normal(rows, cols, dtype=dtype), normal(rows, outer, dtype=dtype, seed=1)
    kept = ops.op_checkpoint(x)
    got = ops.op_checkpoint_product(g, kept)
    v = ops.op_restore(kept).double()
    want, size = g.double().t().contiguous() @ v, g.double().abs().t().contiguous() @ v.abs()
    assert got.shape == (outer, cols) and got.dtype is dtype
    close(got, want, gamma(rows) * size + half_step(dtype) * want.abs() + least(dtype), "product")


# ---- layer norm ----
NORM_SHAPES = [(1, 1), (3, 8), (1, 96), (70, 96), (5, 128), (9, 131), (33, 256), (4, 257), (13, 511), (37, 771), (130, 1024), (6, 1280), (5, 2048),
               (3, 2053), (3, 4096), (2, 5000), (2, 8192), (2, 8200), (1, 16384)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_layer_norm(rows, cols, dtype):
    eps = 1e-5
    x = (normal(rows, cols) * 2 + normal(rows, 1, seed=3)).to(dtype).requires_grad_()
    w, b = (1 + 0.1 * normal(cols, seed=4)).to(dtype).requires_grad_(), normal(cols, dtype=dtype, seed=5).requires_grad_()
    dy = normal(rows, cols, dtype=dtype, seed=6)
    y = ops.op_layer_norm(x, w, b, eps)
    with torch.no_grad():
        assert torch.equal(ops.op_layer_norm(x, w, b, eps), y)
    codes, scale, mn = ops.op_checkpoint(x)[:3]      # what the forward pass keeps, made by itself
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy)
    X, W, B, DY = (t.detach().double() for t in (x, w, b, dy))
    tiny = least(dtype)
    h, gm = half_step(dtype), gamma(cols)
    mean, var = X.mean(1, keepdim=True), X.var(1, unbiased=False, keepdim=True)
    rstd = (var + eps).rsqrt()
    d_mean = gm * X.abs().mean(1, keepdim=True)
    # relative: the variance's own sum, the square of the mean's error, the root and the quotient
    d_rstd = gm + d_mean ** 2 * rstd ** 2 + 2 * rstd * rstd * d_mean * (X - mean).abs().mean(1, keepdim=True) + 4 * U
    xh = (X - mean) * rstd
    d_xh = rstd * (d_mean + U * X.abs() + U * mean.abs()) + xh.abs() * (d_rstd + 4 * U)
    want = xh * W + B
    close(y.detach(), want, d_xh * W.abs() + 2 * U * (want.abs() + B.abs()) + h * want.abs() + tiny, "y")
    v, off = values_of(codes, scale, mn, cols)
    xh = (v - mean) * rstd
    d_xh = rstd * (d_mean + off + U * (v.abs() + mean.abs())) + xh.abs() * (d_rstd + 4 * U)
    g = DY * W
    mgx = (g * xh).mean(1, keepdim=True)
    want = rstd * (g - g.mean(1, keepdim=True) - xh * mgx)
    size = g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True)
    bound = rstd * ((gm + d_rstd + 8 * U) * size + d_xh * mgx.abs() + xh.abs() * (g.abs() * d_xh).mean(1, keepdim=True))
    close(dx, want, bound + h * want.abs() + tiny, "dx")
    want = (DY * xh).sum(0)
    close(dw, want, (DY.abs() * d_xh).sum(0) + gamma(rows) * (DY * xh).abs().sum(0) + h * want.abs() + tiny, "dw")
    want = DY.sum(0)
    close(db, want, gamma(rows) * DY.abs().sum(0) + h * want.abs() + tiny, "db")


@pytest.mark.parametrize("with_weight,with_bias", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weight_or_bias(with_weight, with_bias):
    x = normal(50, 200).requires_grad_()
    w = normal(200, seed=2).requires_grad_() if with_weight else None
    b = normal(200, seed=3).requires_grad_() if with_bias else None
    full_w = w if with_weight else torch.ones(200, device="cuda", requires_grad=True)
    full_b = b if with_bias else torch.zeros(200, device="cuda", requires_grad=True)
    dy = normal(50, 200, seed=4)
    y, z = ops.op_layer_norm(x, w, b), ops.op_layer_norm(x, full_w, full_b)
    assert torch.equal(y, z)
    wanted = [x] + [t for t in (w, b) if t is not None]
    for got, want in zip(torch.autograd.grad(y, wanted, dy), torch.autograd.grad(z, wanted, dy)):
        assert torch.equal(got, want)


def test_layer_norm_of_many_rows_adds_up_every_one():
    """More rows than the backward pass has workgroups, in every shape of a row."""
    for rows, cols in ((40000, 16), (20000, 200), (9000, 400), (3000, 1200)):
        x = normal(rows, cols).requires_grad_()
        w, b = torch.ones(cols, device="cuda", requires_grad=True), torch.zeros(cols, device="cuda", requires_grad=True)
        dy = (torch.arange(rows, device="cuda") % 2).float().unsqueeze(1).expand(rows, cols)
        db, = torch.autograd.grad(ops.op_layer_norm(x, w, b), [b], dy)
        assert torch.equal(db, torch.full_like(db, float(rows // 2)))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,outer,cols", [(64, 64, 640), (300, 300, 1032), (200, 1300, 2056), (50, 4096, 4096)])
def test_checkpoint_product_has_the_values_that_restore_gives(rows, outer, cols, dtype):
    """Rows of the unit matrix pick values one by one: a value rounded in another way than op_restore rounds it is seen."""
    c = ops.op_checkpoint(normal(rows, cols, dtype=dtype))
    got = ops.op_checkpoint_product(torch.eye(rows, outer, dtype=dtype, device="cuda"), c)
    assert torch.equal(got[:rows], ops.op_restore(c)) and not got[rows:].any()


# ---- linear layers ----
def kept_activation(x, w, b, act):
    """Codes, scale and min of x w^T + b as the forward pass keeps them: the same call of the library, on rows of whole 16-byte pieces."""
    rows, inner, outer = x.shape[0], x.shape[1], w.shape[0]
    whole = (inner + 7) // 8 * 8
    x, w = (torch.nn.functional.pad(t, (0, whole - inner)).contiguous().clone() for t in (x, w))
    codes = torch.zeros(rows, (outer + 15) // 16 * 16, dtype=torch.int8, device="cuda")
    scale, mn = (torch.zeros(rows, (outer + 255) // 256, device="cuda") for _ in range(2))
    y = torch.empty(rows, outer, dtype=x.dtype, device="cuda")
    ws = torch.empty(_abi.lib().gact_linear_workspace_bytes(_abi.dtype_code(x.dtype), rows, whole, outer, 1) + 16, dtype=torch.uint8, device="cuda")
    _abi.check(_abi.lib().gact_linear(x.data_ptr(), whole, w.data_ptr(), whole, _abi.ptr(b), None, 0, {"gelu": 1, "gelu_tanh": 2, "silu": 3}[act],
                                      _abi.dtype_code(x.dtype), rows, whole, outer, y.data_ptr(), codes.data_ptr(), codes.stride(0),
                                      scale.data_ptr(), mn.data_ptr(), _abi.ptr(ws), _abi.stream_of(x)))
    return codes, scale, mn


def check_linear(rows, inner, outer, dtype, act, with_bias, with_residual, view=lambda t: t):
    x, w = view(normal(rows, inner, dtype=dtype)).requires_grad_(), view(normal(outer, inner, dtype=dtype, seed=1, scale=inner ** -0.5)).requires_grad_()
    b = normal(outer, dtype=dtype, seed=2).requires_grad_() if with_bias else None
    r = view(normal(rows, outer, dtype=dtype, seed=3)).requires_grad_() if with_residual else None
    dy = view(normal(rows, outer, dtype=dtype, seed=4))
    tiny, h = least(dtype), half_step(dtype)
    X, W, DY = x.detach().double(), w.detach().double(), dy.double()
    B = b.detach().double() if with_bias else torch.zeros(outer, dtype=torch.float64, device="cuda")
    R = r.detach().double() if with_residual else torch.zeros(1, 1, dtype=torch.float64, device="cuda")
    z = X @ W.t().contiguous() + B
    d_z = gamma(inner) * (X.abs() @ W.abs().t().contiguous() + B.abs())
    want = activation(z, act)[0] + R
    fn = FUNCTION if act else 0.0
    bound = MAX_SLOPE * d_z + fn * (1 + z.abs()) + 2 * U * (want.abs() + R.abs()) + h * want.abs() + tiny
    with torch.no_grad():
        close(ops.op_linear(x, w, b, act, r), want, bound, "y without gradient")
    y = ops.op_linear(x, w, b, act, r)
    close(y.detach(), want, bound, "y")
    kept = ops.op_restore(ops.op_checkpoint(x)).double()
    dz, d_dz = DY, torch.zeros_like(DY)
    if act:
        saved = kept_activation(x.detach(), w.detach(), b, act)
        v, off = values_of(*saved, outer)
        close(v, z, 0.5001 / spread(saved[1], outer).double() + 2 * d_z + off + 2 * U * z.abs() + 4e-6 / 255, "codes of z")
        slope = activation(v, act)[1]
        dz = DY * slope
        d_dz = DY.abs() * (FUNCTION + MAX_SLOPE * off) + 2 * U * dz.abs()
    rounded = (h * dz.abs() + tiny if act else 0) + d_dz        # dz enters the products in the layer's type
    wanted = [t for t in (x, w, b, r) if t is not None]
    grads = dict(zip([n for n, t in zip("xwbr", (x, w, b, r)) if t is not None], torch.autograd.grad(y, wanted, dy)))
    want = dz @ W
    rounded = rounded if act else torch.zeros_like(dz)
    close(grads["x"], want, rounded @ W.abs() + gamma(outer) * (dz.abs() @ W.abs()) + h * want.abs() + tiny, "dx")
    want = dz.t().contiguous() @ kept
    close(grads["w"], want, rounded.t().contiguous() @ kept.abs() + gamma(rows) * (dz.abs().t().contiguous() @ kept.abs()) + h * want.abs() + tiny, "dw")
    if with_bias:
        want = dz.sum(0)
        close(grads["b"], want, d_dz.sum(0) + gamma(rows) * dz.abs().sum(0) + h * want.abs() + tiny, "db")
    if with_residual:
        assert torch.equal(grads["r"], dy)


LINEAR_SHAPES = [(1, 1, 1), (1, 64, 16), (3, 9, 5), (16, 256, 48), (17, 100, 33), (33, 264, 40), (64, 520, 257), (65, 128, 128), (100, 771, 130),
                 (129, 64, 384), (200, 1000, 263), (260, 320, 520), (1030, 136, 516), (5000, 24, 96), (700, 16, 125)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,inner,outer", LINEAR_SHAPES)
def test_linear(rows, inner, outer, dtype):
    for n, (act, with_bias, with_residual) in enumerate(itertools.product((None, "gelu", "gelu_tanh", "silu"), (True, False), (False, True))):
        if rows > 64 and n % 3:         # every activation, with and without either operand, in turn
            continue
        check_linear(rows, inner, outer, dtype, act, with_bias, with_residual)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
def test_linear_of_many_tiles(dtype):
    """Enough of them for the largest tiles, none of whose edges the sizes meet."""
    check_linear(4200, 136, 4104, dtype, "gelu", True, True)
    check_linear(4099, 200, 4099, dtype, "silu", True, False)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,inner,outer", [(1, 4096, 264), (24, 2056, 264), (64, 4100, 72), (65, 1030, 48), (100, 2104, 520), (300, 4000, 130),
                                              (50, 4096, 4096), (20, 2047, 4100)])
def test_linear_cut_along_its_depth(rows, inner, outer, dtype):
    for act, with_bias, with_residual in ((None, True, True), ("gelu", True, False), ("silu", False, True)):
        check_linear(rows, inner, outer, dtype, act, with_bias, with_residual)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_linear_of_strided_operands(dtype):
    def wider(t):       # rows of a wider matrix, at an address that no piece begins at
        base = torch.empty(t.shape[0], t.shape[1] + 13, dtype=t.dtype, device=t.device)
        base[:, 5:5 + t.shape[1]] = t
        return base[:, 5:5 + t.shape[1]].detach()

    def aligned_wider(t):
        base = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=t.device)
        base[:, 8:8 + t.shape[1]] = t
        return base[:, 8:8 + t.shape[1]].detach()

    for view in (wider, aligned_wider, lambda t: t.t().contiguous().t().detach()):
        check_linear(70, 264, 136, dtype, "gelu", True, True, view)
        check_linear(9, 40, 24, dtype, None, True, True, view)


def test_linear_gradients_by_differences():
    """The derivative along random directions, from float32 outputs far apart enough for their rounding."""
    x, w, b = normal(80, 96), normal(64, 96, seed=1, scale=0.1), normal(64, seed=2)
    dy = normal(80, 64, seed=3)
    for act in (None, "gelu", "gelu_tanh", "silu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(ops.op_linear(*leaves, act), leaves, dy)
        for n, name in enumerate(("x", "w", "b")):
            way = normal(*leaves[n].shape, seed=9 + n)
            step = 1e-2

            def out(s):
                moved = [t.detach() + (s * way if k == n else 0) for k, t in enumerate(leaves)]
                with torch.no_grad():
                    return (ops.op_linear(*moved, act).double() * dy.double()).sum()

            numeric = (out(step) - out(-step)) / (2 * step)
            analytic = (grads[n].double() * way.double()).sum()
            # 5120 outputs with independent errors: a code of x (about 1/50 of its deviation) or z moves a term by a percent
            scale = (grads[n].double().norm() * way.double().norm())
            assert abs(numeric - analytic) < 0.01 * scale, (act, name, float(numeric), float(analytic), float(scale))


def test_empty_rows():
    w, b = normal(32, 16).requires_grad_(), normal(32).requires_grad_()
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = ops.op_linear(x, w, b, "gelu")
    assert y.shape == (0, 32)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.empty(0, 32, device="cuda"))
    assert dx.shape == (0, 16) and not dw.any() and not db.any()
    nw, nb = torch.ones(16, device="cuda", requires_grad=True), torch.ones(16, device="cuda", requires_grad=True)
    y = ops.op_layer_norm(x, nw, nb)
    dx, dw, db = torch.autograd.grad(y, [x, nw, nb], torch.empty(0, 16, device="cuda"))
    assert y.shape == dx.shape == (0, 16) and not dw.any() and not db.any()
    kept = ops.op_checkpoint(x)
    assert ops.op_restore(kept).shape == (0, 16)
    assert not ops.op_checkpoint_product(torch.empty(0, 8, device="cuda"), kept).any()


def test_unfinite_inputs_stay_where_they_are():
    """An infinity or a NaN in a row is in that row's results only, and in the weight's gradient."""
    for bad in (float("inf"), float("nan")):
        x = normal(40, 300, dtype=torch.bfloat16)
        x[7, 3] = bad
        w = normal(64, 300, dtype=torch.bfloat16, seed=1, scale=0.05)
        with torch.no_grad():
            y = ops.op_linear(x, w)
            n = ops.op_layer_norm(x)
        for out in (y, n):
            finite = torch.isfinite(out).all(1)
            assert not finite[7] and finite.sum() == 39


def test_refusals():
    x, w = normal(8, 16), normal(4, 16, seed=1)
    with pytest.raises(RuntimeError, match="unknown activation"):
        ops.op_linear(x, w, None, "relu")
    with pytest.raises(RuntimeError, match="type of weight"):
        ops.op_linear(x, w.half())
    with pytest.raises(RuntimeError, match="weight must be"):
        ops.op_linear(x, normal(4, 17))
    with pytest.raises(RuntimeError, match="dimension of bias"):
        ops.op_linear(x, w, normal(5))
    with pytest.raises(RuntimeError, match="residual"):
        ops.op_linear(x, w, None, None, normal(8, 5))
    with pytest.raises(RuntimeError, match="type of data"):
        ops.op_linear(x.double(), w.double())
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.op_linear(x, w.cpu())
    with pytest.raises(RuntimeError, match="columns"):
        ops.op_layer_norm(torch.zeros(1, 16385, device="cuda"))
    with pytest.raises(RuntimeError, match="dimension of weight"):
        ops.op_layer_norm(x, normal(8))
    with pytest.raises(RuntimeError, match="type of data"):
        ops.op_checkpoint(x.int())
    kept = ops.op_checkpoint(x)
    with pytest.raises(RuntimeError, match="rows"):
        ops.op_checkpoint_product(normal(7, 4), kept)
    with pytest.raises(RuntimeError, match="do not belong"):
        ops.op_restore(kept._replace(shape=(8, 17)))
    with pytest.raises(RuntimeError, match="do not belong"):
        ops.op_checkpoint_product(normal(8, 4), kept._replace(codes=kept.codes[:4]))
    with pytest.raises(TypeError):
        ops.op_restore([kept.codes, 8, kept.scale, kept.min])
