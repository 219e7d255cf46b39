"""Attention and its gradients on the GPU against the formulas in 64 bits; the bounds are worked out element by element in attention_reference.py."""
import math

import pytest
import torch

from gact import ops
from attention_reference import attend
from layer_reference import close

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None  # noqa: E731


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


def inputs(b, h, g, m, n, w, dtype, bias=False, mask=False, scale=1.0):
    q, k, v = normal(b, h, m, w, dtype=dtype, scale=scale), normal(b, g, n, w, dtype=dtype, seed=1), normal(b, g, n, w, dtype=dtype, seed=2)
    there = None
    if mask:
        there = torch.rand(b, n, generator=torch.Generator().manual_seed(3)).cuda() < 0.7
        there[0, n // 2:] = False
    return q, k, v, normal(b, h, m, w, dtype=dtype, seed=4), normal(h, max(m + n - 1, 0), seed=5) if bias else None, there


def check(q, k, v, dy, bias, mask, causal=False, scale=None, train=True):
    leaves = [t.detach().requires_grad_(train) for t in (q, k, v) + ((bias,) if bias is not None else ())]
    y = ops.op_attention(*leaves[:3], leaves[3] if bias is not None else None, mask, causal, scale)
    want = attend(q, k, v, dy if train else None, bias, mask, causal, scale)
    assert y.shape == q.shape and y.dtype is q.dtype
    close(y, *want["y"], "y")
    if not train:
        return y
    with torch.no_grad():
        assert torch.equal(ops.op_attention(q, k, v, bias, mask, causal, scale), y)
    grads = torch.autograd.grad(y, leaves, dy)
    for name, leaf, grad in zip(("dq", "dk", "dv", "dbias"), leaves, grads):
        assert grad.shape == leaf.shape and grad.dtype is leaf.dtype
        close(grad, *want[name], name)
    return y, grads


# batch, heads, key heads, queries, keys, width
SHAPES = [(1, 1, 1, 1, 1, 1), (1, 1, 1, 1, 1, 64), (2, 3, 3, 32, 32, 32), (1, 2, 2, 33, 31, 64), (2, 2, 1, 64, 64, 128), (1, 4, 2, 65, 63, 96), (3, 2, 2, 49, 49, 32),
          (1, 3, 3, 128, 200, 64), (2, 6, 2, 197, 77, 72), (1, 2, 2, 129, 257, 7), (1, 1, 1, 300, 5, 40), (1, 8, 2, 5, 300, 64), (1, 2, 2, 260, 321, 128), (2, 1, 1, 7, 1, 13)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["plain", "causal", "mask", "bias", "all"])
def test_attention(shape, kind, dtype):
    q, k, v, dy, bias, mask = inputs(*shape, dtype, kind in ("bias", "all"), kind in ("mask", "all"))
    check(q, k, v, dy, bias, mask, kind in ("causal", "all"))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 4097, 64), (24, 4, 4, 1, 517, 64), (1, 32, 8, 1, 9000, 128), (2, 8, 1, 4, 1025, 80), (1, 2, 1, 100, 2000, 32),
                                   (1, 1, 1, 31, 128, 128), (2, 2, 2, 1, 257, 5), (1, 1, 1, 32, 40000, 128), (1, 16, 1, 3, 2048, 96)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["plain", "all"])
def test_few_queries_behind_many_keys(shape, kind, dtype):
    q, k, v, dy, bias, mask = inputs(*shape, dtype, kind == "all", kind == "all")
    check(q, k, v, dy, bias, mask, kind == "all", train=False)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1, 4, 2, 3, 3000, 64), (2, 2, 2, 1, 700, 128)], ids=lambda s: "x".join(map(str, s)))
def test_few_queries_train(shape, dtype):
    q, k, v, dy, bias, mask = inputs(*shape, dtype, True, True)
    check(q, k, v, dy, bias, mask, True)


# up to 64 queries and keys, of one head or of several that share its keys
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(2, 3, 3, 64, 64, 64), (3, 6, 2, 40, 64, 64), (2, 4, 1, 64, 17, 80), (1, 2, 2, 5, 60, 32), (2, 8, 1, 33, 33, 128), (30, 3, 3, 49, 49, 32),
                                   (1, 4, 2, 31, 33, 100), (256, 4, 2, 33, 35, 40), (520, 3, 1, 5, 64, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["plain", "causal", "mask", "both"])
def test_short_sequences(shape, kind, dtype):
    q, k, v, dy, bias, mask = inputs(*shape, dtype, False, kind in ("mask", "both"))
    check(q, k, v, dy, bias, mask, kind in ("causal", "both"))


# the batch entries' diagonals are added up by several waves where there are few blocks of queries
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(37, 2, 2, 20, 24, 64), (300, 1, 1, 54, 54, 128), (21, 2, 1, 100, 40, 32), (9, 2, 2, 230, 70, 32)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["bias", "all"])
def test_biases_of_many_batch_entries(shape, kind, dtype):
    q, k, v, dy, bias, mask = inputs(*shape, dtype, True, kind == "all")
    check(q, k, v, dy, bias, mask, kind == "all")


# few tiles, with the keys and the queries cut into splits whose sums are added afterwards
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(1, 1, 1, 700, 900, 64), (1, 4, 1, 333, 1100, 128), (2, 2, 2, 1500, 130, 40), (1, 2, 2, 130, 2049, 96), (1, 1, 1, 1025, 513, 32),
                                   (3, 4, 2, 40, 650, 77)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["plain", "causal", "mask", "all"])
def test_gradients_of_few_tiles(shape, kind, dtype):
    q, k, v, dy, bias, mask = inputs(*shape, dtype, kind == "all", kind in ("mask", "all"))
    check(q, k, v, dy, bias, mask, kind in ("causal", "all"))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_queries_that_see_nothing(dtype):
    q, k, v, dy, bias, _ = inputs(3, 2, 2, 70, 40, 64, dtype, True)
    mask = torch.ones(3, 40, dtype=torch.bool, device="cuda")
    mask[1] = False
    mask[2, 1:] = False
    # causal, with fewer keys than queries: the first 30 queries of each see nothing either
    y, (dq, dk, dv, dbias) = check(q, k, v, dy, bias, mask, True)
    assert not y[1].any() and not y[:, :, :30].any() and not dq[1].any() and not dq[:, :, :30].any() and not dk[1].any() and not dv[1].any()
    assert not dk[2, :, 1:].any() and not dv[2, :, 1:].any() and y[0, :, 30:].any()
    single = ops.op_attention(q[:, :, :1], k, v, None, torch.zeros_like(mask))
    assert not single.any()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m", [1, 90])
def test_absent_keys_hold_anything(dtype, m):
    q, k, v, dy, bias, mask = inputs(2, 4, 2, m, 300, 64, dtype, True, True)
    clean = [t.clone() for t in (k, v)]
    for n, t in enumerate((k, v)):
        t.transpose(1, 2)[~mask] = (math.nan, math.inf)[n]
    k[0, 0, 299], v[0, 1, 299] = -math.inf, math.nan
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    y = ops.op_attention(*leaves[:3], bias, mask, True)
    grads = torch.autograd.grad(y, leaves, dy)
    others = [t.detach().requires_grad_() for t in (q, *clean, bias)]
    same = ops.op_attention(*others[:3], others[3], mask, True)
    assert torch.equal(y, same)
    for a, b in zip(grads, torch.autograd.grad(same, others, dy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("m,n", [(1, 600), (80, 80)])
def test_biases_that_hide(dtype, m, n):
    q, k, v, dy, bias, _ = inputs(2, 2, 2, m, n, 32, dtype, True)
    bias[0, ::3] = -math.inf
    bias[0, 1::3] = torch.finfo(torch.float32).min
    bias[1, : (m + n) // 2] = -1e30
    check(q, k, v, dy, bias, None)
    bias[:] = torch.finfo(torch.float32).min
    y, grads = check(q, k, v, dy, bias, None)
    assert not y.any() and not any(g.any() for g in grads)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_large_scores(dtype):
    """One key has all of the probability; scores far apart, rising along the keys so that the maximum moves with every tile."""
    q, k, v, dy, _, _ = inputs(1, 2, 2, 64, 500, 64, dtype, scale=4.0)
    k *= torch.linspace(0.1, 4, 500, device="cuda")[:, None].to(dtype)
    check(q, k, v, dy, None, None)
    check(q, k, v, dy, None, None, scale=1.0)
    check(q[:, :, :1], k, v, dy[:, :, :1], None, None, scale=1.0)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_nan_and_infinity_show_where_they_are(dtype):
    q, k, v, dy, _, _ = inputs(2, 2, 2, 70, 70, 64, dtype)
    q[0, 1, 5, 3], q[1, 0, 7, 0] = math.nan, math.inf
    y = ops.op_attention(q, k, v)
    bad = ~torch.isfinite(y).all(3)
    assert bad[0, 1, 5] and bad[1, 0, 7] and int(bad.sum()) == 2
    v[0, 0, 3, 3] = math.nan
    y = ops.op_attention(q, k, v)
    assert torch.isnan(y[0, 0, :, 3]).all() and torch.isfinite(y[0, 0, :, :3]).all() and torch.isfinite(y[1, 1]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=ids)
@pytest.mark.parametrize("apart", [False, True])
def test_what_the_results_rounding_leaves_out_counts_in_the_gradients(dtype, apart):
    """Two keys of one score, values one step apart: the result lies in the middle, ds is half a step, and a rounded result would make it none or a whole one."""
    step = torch.finfo(dtype).eps
    m = 1 if apart else 64
    q, k = torch.zeros(1, 1, m, 64), torch.zeros(1, 1, 2, 64)
    k[0, 0, 0, 0], k[0, 0, 1, 0] = 1.0, 1.0
    k[0, 0, 0, 1], k[0, 0, 1, 1] = 1.0, -1.0
    v = torch.ones(1, 1, 2, 64)
    v[0, 0, 0] += step
    q, k, v = (t.to(dtype).cuda() for t in (q, k, v))
    q.requires_grad_()
    dy = torch.ones(1, 1, m, 64, dtype=dtype, device="cuda")
    y = ops.op_attention(q, k, v, scale=1.0)
    dq = torch.autograd.grad(y, q, dy)[0].double()
    # ds = +-1/2 * 64 * step / 2, exact in the type but for a 254th of each half step that the bytes round by
    want = 64 * step / 2
    assert (dq[0, 0, :, 1] - want).abs().max() <= want * (1 / 254 + step) and dq[0, 0, :, 0].abs().max() <= want * (1 / 254 + step) * 2


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_strides_views_and_shared_storage(dtype):
    b, m, h, w = 2, 70, 4, 64
    packed = normal(b, m, 3, h, w, dtype=dtype)
    q, k, v = packed.permute(2, 0, 3, 1, 4)
    dy = normal(b, m, h, w, dtype=dtype, seed=1).transpose(1, 2)
    y, _ = check(q, k, v, dy, None, None, True)
    assert y.transpose(1, 2).is_contiguous()
    views = [q.contiguous()[:, :, ::2], q[..., :33], q[..., 1:34], q.transpose(2, 3).contiguous().transpose(2, 3), q[:, :1].expand(b, h, m, w),
             q[:1].expand(b, h, m, w), q[:, :, :1].expand(b, h, m, w), q.flip(2), torch._neg_view(q)]
    for view in views:
        w2 = view.shape[-1]
        plain = view.contiguous().clone()
        other, grad = k[..., :w2], dy[:, :, :view.shape[2], :w2]
        got, want = [], []
        for out, x in ((got, view), (want, plain)):
            leaf = x.detach().requires_grad_() if not x.is_neg() else x
            out.append(ops.op_attention(leaf, other, other, None, None, True))
            out.append(ops.op_attention(other[:, :, :view.shape[2]], leaf, leaf, None, None, True))
        for a, c in zip(got, want):
            assert torch.equal(a, c)
        check(plain, other, other, grad, None, None)
        # a gradient of any layout
        leaf = plain.requires_grad_()
        y = ops.op_attention(leaf, other, other)
        strange = grad.transpose(2, 3).contiguous().transpose(2, 3)
        assert torch.equal(*(torch.autograd.grad(y, leaf, g, retain_graph=True)[0] for g in (grad, strange)))
        ones = torch.autograd.grad(y.sum(), leaf, retain_graph=True)[0]
        assert torch.equal(ones, torch.autograd.grad(y, leaf, torch.ones_like(y))[0])


def test_masks_and_biases_of_any_stride():
    q, k, v, dy, bias, mask = inputs(3, 2, 2, 40, 90, 64, torch.bfloat16, True, True)
    want = ops.op_attention(q, k, v, bias, mask)
    wide = torch.zeros(3, 180, dtype=torch.bool, device="cuda")
    wide[:, ::2] = mask
    assert torch.equal(ops.op_attention(q, k, v, bias, wide[:, ::2]), want)
    assert torch.equal(ops.op_attention(q, k, v, bias.t().contiguous().t(), mask), want)
    assert torch.equal(ops.op_attention(q, k, v, torch._neg_view(-bias), mask), want)
    one = mask[1:2].expand(3, 90)
    assert torch.equal(ops.op_attention(q, k, v, None, one), ops.op_attention(q, k, v, None, one.contiguous()))
    shared = bias[:1].clone().requires_grad_()
    y = ops.op_attention(q, k, v, shared.expand(2, -1), mask)
    each = bias[:1].expand(2, -1).contiguous().requires_grad_()
    grads = torch.autograd.grad(y, shared, dy)[0], torch.autograd.grad(ops.op_attention(q, k, v, each, mask), each, dy)[0]
    assert torch.equal(grads[0], grads[1].sum(0, keepdim=True))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_empty(dtype):
    for b, m, n in ((0, 5, 7), (2, 0, 7), (2, 5, 0), (2, 0, 0), (0, 0, 0)):
        q, k, v = (torch.zeros(s, dtype=dtype, device="cuda").requires_grad_() for s in ((b, 4, m, 64), (b, 2, n, 64), (b, 2, n, 64)))
        bias = torch.zeros(4, max(m + n - 1, 0), device="cuda").requires_grad_()
        with torch.no_grad():
            for t in (q, k, v):
                t += 1
        for causal in (False, True):
            y = ops.op_attention(q, k, v, bias, torch.ones(b, n, dtype=torch.bool, device="cuda"), causal)
            assert y.shape == q.shape and not y.any()
            grads = torch.autograd.grad(y, [q, k, v, bias], torch.ones_like(y))
            assert all(g.shape == t.shape and not g.any() for g, t in zip(grads, (q, k, v, bias)))


def test_gradients_against_differences():
    q, k, v, dy, bias, mask = inputs(1, 4, 2, 9, 11, 16, torch.float32, True, True)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, bias)]
    y = ops.op_attention(*leaves[:3], leaves[3], mask, True)
    grads = torch.autograd.grad(y, leaves, dy)
    step = 2.0 ** -6
    for n in range(4):
        where = normal(*leaves[n].shape, seed=20 + n)

        def at(s):
            moved = [t.detach().double() + (s * where.double() if i == n else 0) for i, t in enumerate(leaves)]
            return (attend(*moved[:3], None, moved[3], mask, True)["y"][0] * dy.double()).sum()

        # four values in 64 bits: the difference's error is of the fourth power of the step, below what 32-bit sums are off by
        slope = (8 * (at(step / 2) - at(-step / 2)) - (at(step) - at(-step))) / (6 * step)
        got, size = (grads[n].double() * where.double()).sum(), (grads[n].double() * where.double()).abs().sum()
        assert abs(got - slope) <= 1e-4 * size + 1e-6


def test_the_same_bits_every_time():
    for dtype in TYPES:
        q, k, v, dy, bias, mask = inputs(4, 8, 2, 300, 500, 64, dtype, True, True)
        leaves = [t.requires_grad_() for t in (q, k, v, bias)]
        first = None
        for _ in range(3):
            y = ops.op_attention(*leaves[:3], bias, mask, True)
            all_of = [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
            first = first or all_of
            assert all(torch.equal(a, b) for a, b in zip(first, all_of))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("shape", [(2, 2, 2, 50, 60, 64), (1, 4, 2, 700, 900, 64), (2, 16, 16, 1100, 1030, 64)], ids=lambda s: "x".join(map(str, s)))
def test_some_of_the_gradients(shape, dtype):
    """A single kernel, splits of either side, and neither: a gradient is the same whichever others are wanted."""
    q, k, v, dy, bias, mask = inputs(*shape, dtype, False, True)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    y = ops.op_attention(*leaves, None, mask, True)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for some in ([0], [1], [2], [0, 2], [1, 2], [2, 0]):
        got = torch.autograd.grad(y, [leaves[n] for n in some], dy, retain_graph=True)
        assert all(torch.equal(g, want[n]) for g, n in zip(got, some))


def test_only_the_gradients_that_are_asked_for():
    q, k, v, dy, bias, mask = inputs(2, 4, 2, 100, 100, 64, torch.bfloat16, True)
    leaves = [t.requires_grad_() for t in (q, k, v, bias)]
    y = ops.op_attention(*leaves[:3], bias)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for n, leaf in enumerate(leaves):
        assert torch.equal(torch.autograd.grad(y, leaf, dy, retain_graph=True)[0], want[n])
    k.requires_grad_(False)
    y = ops.op_attention(q, k, v, bias.detach())
    assert torch.equal(torch.autograd.grad(y, v, dy)[0], want[2])


def test_offsets_past_32_bits():
    """A cache of 2^31 + elements, of which two tokens' heads far apart are looked at."""
    n, w = (1 << 24) - 3, 128
    cache = torch.zeros(1, n, 1, w, dtype=torch.float16, device="cuda")
    cache[0, n - 40:] = normal(40, 1, w, dtype=torch.float16)
    k = cache.transpose(1, 2)
    q = normal(1, 1, 1, w, dtype=torch.float16, seed=1, scale=4)
    mask = torch.zeros(1, n, dtype=torch.bool, device="cuda")
    mask[0, n - 40:] = True
    got = ops.op_attention(q, k, k, None, mask)
    assert torch.equal(got, ops.op_attention(q, k, k, None, mask, True))
    tail = k[:, :, n - 40:].contiguous()
    close(got, *attend(q, tail, tail)["y"], "y")
    # batch entries and heads that lie far apart
    far = torch.zeros(2, 40, (1 << 31) // 80 // 64 + 1, 64, dtype=torch.float16, device="cuda")
    near = normal(2, 40, 1, 64, dtype=torch.float16, seed=2)
    far[:, :, -1:] = near
    rows = far[:, :, -1:].transpose(1, 2)
    assert rows.stride(0) > 1 << 30
    assert torch.equal(ops.op_attention(rows, rows, rows), ops.op_attention(*[near.transpose(1, 2)] * 3))


def test_many_heads_and_batch_entries():
    q, k, v, dy, _, _ = inputs(70000, 1, 1, 2, 2, 8, torch.float32)
    check(q, k, v, dy, None, None)
