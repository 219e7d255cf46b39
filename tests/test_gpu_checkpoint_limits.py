"""The layers on 8-bit checkpoints at their limits: launches of 2^32 threads and more, the largest values."""
import pytest
import torch
import torch.nn.functional as F

from gact import ops
from gact.cpp_extension import _abi

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _give_memory_back():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def repeated(rows, cols, dtype, period):
    """[rows, cols] of which every `period` rows are the same, and those rows."""
    g = torch.Generator(device="cuda").manual_seed(rows % 1000 + cols)
    small = torch.randn(period, cols, generator=g, device="cuda").to(dtype)
    x = torch.empty(rows, cols, dtype=dtype, device="cuda")
    x.view(-1, period, cols).copy_(small)
    return x, small


def all_like(big, small):
    """Whether every part of `big` is `small`."""
    return all(bool((part == small).all()) for part in big.view(-1, *small.shape).split(1 << 14))


# threads of the launch over 2^32: (groups / groups of a workgroup) of 256 threads.  Sixteen lanes to a group, then 32 with a short last group
@pytest.mark.parametrize("rows,cols,a_workgroup", [((1 << 28) + 64, 1, 16), ((1 << 26) + 64, 257, 8)])
def test_checkpoint_of_more_groups_than_a_launch_is_wide(rows, cols, a_workgroup):
    assert rows * -(-cols // 256) // a_workgroup * 256 > 1 << 32
    x, small = repeated(rows, cols, torch.float16, 64)
    kept, want = ops.op_checkpoint(x), ops.op_checkpoint(small)
    del x
    assert all_like(kept.codes[:, :cols].contiguous(), want.codes[:, :cols])
    assert all_like(kept.scale, want.scale) and all_like(kept.min, want.min)
    back = ops.op_restore(kept)
    assert all_like(back, ops.op_restore(want))


def test_layer_norm_of_more_rows_than_a_launch_is_wide():
    rows, cols = (1 << 24) + 64, 1025        # 256 threads to a row
    x, small = repeated(rows, cols, torch.bfloat16, 64)
    w, b = torch.linspace(0.5, 2, cols, device="cuda").bfloat16(), torch.linspace(-1, 1, cols, device="cuda").bfloat16()
    with torch.no_grad():
        assert all_like(ops.op_layer_norm(x, w, b), ops.op_layer_norm(small, w, b))


def test_rows_padded_to_more_pieces_than_a_launch_is_wide():
    rows, cols, to = (1 << 23) + 64, 3, 4096
    x, small = repeated(rows, cols, torch.float16, 64)
    out = torch.empty(rows, to, dtype=torch.float16, device="cuda")
    _abi.check(_abi.lib().gact_pad_rows(x.data_ptr(), _abi.dtype_code(x.dtype), rows, cols, cols, out.data_ptr(), to, _abi.stream_of(x)))
    assert all_like(out, torch.nn.functional.pad(small, (0, to - cols)))


@pytest.mark.parametrize("rows,outer", [(3, 264), (40, 264), (200, 264), (700, 2056), (4100, 4104)])
def test_activations_of_the_largest_values(rows, outer):
    """z up to bfloat16's largest value, of either sign: all three activations leave z as it is there, or nothing of it.  Through the kernel of few
    rows, parts, the finishing kernel and the products' own epilogues, with codes and without."""
    x, w = torch.zeros(rows, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(outer, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 2.0 ** 60
    w[:, 0] = torch.tensor([1.75 * 2.0 ** 67, 1.0 * 2.0 ** 67, -1.5 * 2.0 ** 67, 2.0 ** -50, -2.0 ** -50], device="cuda").repeat(-(-outer // 5))[:outer]
    z = (x[0, 0].double() * w[:, 0].double()).expand(rows, outer)
    for act in ("gelu", "gelu_tanh", "silu"):
        with torch.no_grad():
            assert torch.equal(ops.op_linear(x, w, None, act).double(), z.clamp(min=0))
        leaf = w.clone().requires_grad_()
        y = ops.op_linear(x, leaf, None, act)
        assert torch.equal(y.detach().double(), z.clamp(min=0))


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * len(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def test_a_nan_among_numbers_is_kept_as_its_groups_minimum():
    """As op_quantize keeps it; an infinity's group stands for nothing, and so does one of nothing but NaN."""
    nan, inf = float("nan"), float("inf")
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        x = normal(6, 600, dtype=dtype)
        x[1, 3], x[2, 300], x[3, 599], x[4, 256:512], x[5, :2] = nan, inf, -inf, nan, torch.tensor([inf, -inf], dtype=dtype)
        back, clean = ops.op_restore(ops.op_checkpoint(x)), x.clone()
        clean[1, 3] = torch.cat([x[1, :3], x[1, 4:256]]).min()
        want = ops.op_restore(ops.op_checkpoint(clean))
        lost = torch.zeros(6, 600, dtype=torch.bool, device="cuda")
        lost[2, 256:512] = lost[3, 512:] = lost[4, 256:512] = lost[5, :256] = True
        assert torch.equal(back.isnan(), lost) and torch.equal(back[~lost], want[~lost])
        assert back[1, 3] == clean[1, 3]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,outer", [(10, 40), (50, 520), (200, 264), (700, 2056)])
def test_gradients_of_unfinite_inputs(rows, outer, dtype):
    """dx of the other rows does not see them.  dW from a finite dy sees an infinity in its group's columns, a NaN as that group's minimum;
    behind an activation the row's slopes are not known, and every column of dW is lost."""
    w, dy = normal(outer, 300, dtype=dtype, seed=1, scale=0.05), normal(rows, outer, dtype=dtype, seed=2)

    def grads(x, act):
        leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        return torch.autograd.grad(ops.op_linear(leaves[0], leaves[1], None, act), leaves, dy)

    for bad in (float("inf"), float("nan")):
        x = normal(rows, 300, dtype=dtype)
        x[7, 3] = bad
        clean = x.clone()
        clean[7, 3] = torch.cat([x[7, :3], x[7, 4:256]]).min()
        (dx, dw), (want_dx, want_dw) = grads(x, None), grads(clean, None)
        assert torch.equal(dx, want_dx)
        if bad != bad:
            assert torch.equal(dw, want_dw)
        else:
            assert dw[:, :256].isnan().all() and torch.equal(dw[:, 256:], want_dw[:, 256:])
        others = torch.arange(rows, device="cuda") != 7
        for act in ("gelu", "gelu_tanh", "silu"):
            (dx, dw), (want_dx, _) = grads(x, act), grads(clean, act)
            assert torch.equal(dx[others], want_dx[others]) and dx[7].isnan().all() and dw.isnan().all()
        leaves = [t.requires_grad_() for t in (x.clone(), torch.ones(300, dtype=dtype, device="cuda"), torch.zeros(300, dtype=dtype, device="cuda"))]
        dn = normal(rows, 300, dtype=dtype, seed=3)
        dx, dnw, dnb = torch.autograd.grad(ops.op_layer_norm(*leaves), leaves, dn)
        assert dx[7].isnan().all() and dx[others].isfinite().all() and dnw.isnan().all() and dnb.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,outer", [(10, 40), (50, 520), (200, 264), (700, 2056), (4100, 4104)])
def test_infinities_through_an_activation_are_torchs(rows, outer, dtype):
    x, w = normal(rows, 24, dtype=dtype), normal(outer, 24, dtype=dtype, seed=1)
    plain = x.clone()
    x[7, 3] = float("inf")
    z = torch.where(w[:, 3] > 0, float("inf"), -float("inf")).double()
    others = torch.arange(rows, device="cuda") != 7
    for act, of in (("gelu", F.gelu), ("gelu_tanh", lambda v: F.gelu(v, approximate="tanh")), ("silu", F.silu)):
        want = of(z)
        for leaf in (w, w.clone().requires_grad_()):        # codes of z kept, and not
            y = ops.op_linear(x, leaf, None, act).detach()
            assert torch.equal(y[others], ops.op_linear(plain, leaf, None, act).detach()[others])
            assert torch.equal(y[7].isnan(), want.isnan()) and torch.equal(y[7].isposinf(), want.isposinf())


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,inner,outer", [(3, 40, 33), (40, 264, 520), (200, 72, 264), (700, 72, 2057), (4100, 72, 4104)])
def test_results_do_not_depend_on_addresses(rows, inner, outer, dtype):
    """Biases, a norm's weights, residuals and gradients that begin at any element of a larger tensor, or take every second one."""
    x, w = normal(rows, inner, dtype=dtype), normal(outer, inner, dtype=dtype, seed=1, scale=0.1)
    room = normal(2 * outer + 2 * inner + 16, dtype=dtype, seed=4)
    wide = normal(rows, max(inner, outer) + 16, dtype=dtype, seed=2)
    copy = lambda t: t.clone(memory_format=torch.contiguous_format)  # noqa: E731
    for first, step in ((1, 1), (3, 1), (6, 1), (2, 2)):
        b, nw = room[first:first + step * outer:step], room[first + 1:first + 1 + step * inner:step]
        r = dy = wide[:, first:first + outer]
        for act in (None, "gelu"):
            pair = []
            for args in ((b, r, dy), map(copy, (b, r, dy))):
                bias, residual, g = args
                leaves = [x.clone().requires_grad_(), w.clone().requires_grad_(), bias.detach().requires_grad_()]
                y = ops.op_linear(*leaves, act, residual)
                with torch.no_grad():
                    pair.append([y.detach(), ops.op_linear(x, w, bias, act), ops.op_linear(x, w, bias, act, residual)])
                pair[-1] += torch.autograd.grad(y, leaves, g)
            assert all(torch.equal(a, c) for a, c in zip(*pair)), (first, step, act)
        pair = []
        n = wide[:, first:first + inner]
        for args in ((n, nw, b[:1].expand(inner), n), map(copy, (n, nw, b[:1].expand(inner), n))):
            leaves = [t.detach().requires_grad_() for t in args]
            y = ops.op_layer_norm(*leaves[:3])
            pair.append([y.detach()] + list(torch.autograd.grad(y, leaves[:3], leaves[3].detach())))
        assert all(torch.equal(a, c) for a, c in zip(*pair)), (first, step)
