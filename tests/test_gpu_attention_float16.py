"""Attention's gradients in float16 where ds and probabilities are small, large or far apart: in whichever range, what they are off by stays near the rounding
of the results themselves.

Results are compared by their norms with 64 bits.  A result's rounding is half a step at most, 2^-11 of it or 2^-25.  What else there is of dq and dk: ds as a
pair of float16 numbers, off by 2^-19 of a row's largest or 2^-40; the byte of each o, 2^-19 of do.o; probabilities from scores in 32 bits, 2^-19: of
each ds, together below 2^-17.  A row of dq adds up ds of either sign whose sizes are those of the sum times the root of their number at most, whose
deviation from the mean of k is of order one: 2^-13 of the norm is four times more than that for the widest cancellation here (16).  dv is a
product of probabilities rounded to float16, each off by 2^-11 of itself with a sign of its own."""
import math

import pytest
import torch

from attention_reference import attend
from gact import ops

pytestmark = pytest.mark.gpu

HALF = torch.float16


def normal(*shape, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(HALF).cuda()


def inputs(b, h, g, m, n, w, dy):
    return normal(b, h, m, w), normal(b, g, n, w, seed=1), normal(b, g, n, w, seed=2), normal(b, h, m, w, seed=3, scale=dy)


def own_rounding(x):
    return (2.0 ** -11 * x.abs()).clamp(min=2.0 ** -25).norm()


def check(q, k, v, dy, bias=None, mask=None, causal=False):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    y = ops.op_attention(*leaves, bias, mask, causal)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(y, leaves, dy)))
    want = attend(q, k, v, dy, bias, mask, causal)
    for name in ("dq", "dk"):
        x = want[name][0]
        off = (got[name].double() - x).norm()
        print(name, float(off / x.norm()), float(own_rounding(x) / x.norm()))
        assert torch.isfinite(got[name]).all() and off <= own_rounding(x) + 2.0 ** -13 * x.norm(), name
    # each probability's rounding times dy, added up as roots of squares
    K, V = (t.double().repeat_interleave(q.shape[1] // k.shape[1], 1) for t in (k, v))
    s = q.double() @ K.mT.contiguous() / math.sqrt(q.shape[3])
    i, j = torch.arange(q.shape[2], device="cuda")[:, None], torch.arange(k.shape[2], device="cuda")[None]
    if bias is not None:
        s = s + bias.double()[:, j - i + q.shape[2] - 1]
    hidden = torch.zeros_like(s, dtype=torch.bool)
    if mask is not None:
        hidden |= ~mask[:, None, None, :]
    if causal:
        hidden |= j > i + k.shape[2] - q.shape[2]
    p = torch.softmax(s.masked_fill(hidden, -math.inf), 3).nan_to_num(0.0)
    each = (p.square().mT.contiguous() @ dy.double().square()).view(k.shape[0], k.shape[1], -1, *k.shape[2:]).sum(2).sqrt()
    x = want["dv"][0]
    off = (got["dv"].double() - x).norm()
    print("dv", float(off / x.norm()), float(own_rounding(x) / x.norm()), float(2.0 ** -11 * each.norm() / x.norm()))
    assert off <= own_rounding(x) + 2.0 ** -11 * each.norm() + 2.0 ** -13 * x.norm()


# tiles, splits of either side, one workgroup's keys in turn, rows of every width, one kernel for short sequences, shared key heads
SHAPES = [(1, 2, 2, 1024, 4096, 64), (1, 4, 1, 333, 1100, 128), (2, 6, 2, 200, 771, 72), (1, 3, 3, 700, 650, 32), (64, 8, 8, 260, 256, 64), (16, 16, 8, 300, 300, 128),
          (8, 6, 3, 60, 64, 64), (520, 4, 2, 64, 50, 32), (3, 4, 4, 33, 64, 128), (2, 2, 1, 20, 17, 96)]


@pytest.mark.parametrize("size", [1e-3, 1e-4, 2e-5, 1.0, 1e3])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gradients_of_every_size(shape, size):
    check(*inputs(*shape, size))


@pytest.mark.parametrize("shape", [(2, 4, 2, 700, 900, 64), (1, 2, 2, 260, 321, 128), (4, 4, 4, 40, 64, 64)], ids=lambda s: "x".join(map(str, s)))
def test_small_gradients_with_a_bias_a_mask_and_causal(shape):
    q, k, v, dy = inputs(*shape, 1e-4)
    bias = normal(shape[1], shape[3] + shape[4] - 1, seed=5).float()
    mask = torch.rand(shape[0], shape[4], generator=torch.Generator().manual_seed(3)).cuda() < 0.7
    mask[:, 0] = True
    check(q, k, v, dy, bias, mask, True)
    check(q, k, v, dy, None, mask, True)


def test_probabilities_of_many_keys():
    check(*inputs(1, 1, 1, 64, 300000, 64, 1.0))
    check(*inputs(1, 2, 1, 150, 100001, 96, 0.02))


@pytest.mark.parametrize("shape", [(2, 2, 2, 64, 8, 64), (2, 2, 2, 200, 20, 64), (1, 2, 1, 300, 12, 128)], ids=lambda s: "x".join(map(str, s)))
def test_ds_beyond_float16s_largest(shape):
    """Sums that float16 holds, of products that it does not."""
    q, k, v, dy = inputs(*shape, 1000.0)
    check(q / 64, k / 64, 64 * v, dy)


@pytest.mark.parametrize("shape", [(1, 2, 2, 300, 700, 64), (1, 2, 1, 260, 520, 128), (4, 2, 2, 64, 64, 64)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("side", ["keys", "queries"])
@pytest.mark.parametrize("up", [False, True], ids=["falling", "rising"])
def test_ds_that_differ_by_powers_of_two_along_a_row(shape, side, up):
    """From tile to tile by 2^6 and more, so that what has been added up changes its scale several times, or the small ones come after the large ones."""
    q, k, v, dy = inputs(*shape, 1.0)
    n = shape[4] if side == "keys" else shape[3]
    size = torch.exp2(torch.linspace(-14, 8, n)).cuda()[:, None]
    size = (size if up else size.flip(0)).to(HALF)
    if side == "keys":
        v = v * size
    else:
        dy = dy * size
    check(q, k, v, dy)


@pytest.mark.parametrize("shape", [(1, 2, 2, 300, 400, 64), (1, 2, 2, 200, 130, 128), (2, 2, 2, 64, 64, 64)], ids=lambda s: "x".join(map(str, s)))
def test_an_infinite_gradient_stays_in_its_row(shape):
    q, k, v, dy = inputs(*shape, 1e-3)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    y = ops.op_attention(*leaves)
    want = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for bad in (math.inf, math.nan):
        other = dy.clone()
        other[0, 1, 5, 3] = bad
        dq, dk, dv = torch.autograd.grad(y, leaves, other, retain_graph=True)
        assert not torch.isfinite(dq[0, 1, 5]).any() and not torch.isfinite(dk[0, 1]).any() and not torch.isfinite(dv[0, 1, :, 3]).any()
        there = torch.ones(shape[:2] + shape[3:4], dtype=torch.bool, device="cuda")
        there[0, 1, 5] = False
        assert torch.equal(dq[there], want[0][there]) and torch.equal(dk[0, 0], want[1][0, 0])
        dv[0, 1, :, 3] = want[2][0, 1, :, 3]
        off = (dv[0, 1] - want[2][0, 1]).double()
        assert torch.equal(dv[0, 0], want[2][0, 0]) and torch.isfinite(off).all() and off.abs().max() == 0


@pytest.mark.parametrize("keys,below", [(100000, 32.49), (20000, 8.49), (1000000, 300.49)])
@pytest.mark.parametrize("shape", [(300, 33), (1, 1), (2, 300)], ids=["tiles", "one", "few"])
def test_many_small_probabilities_beside_a_large_one(shape, keys, below):
    """One key's score is so far above all others' that their probabilities, unnormalised, lie between two of float16's subnormal numbers; together they count.
    Each is off by 2^-32 of the largest at most, which one is 1 or more: keys times that of the sum, and of the values' sizes."""
    heads, queries = shape
    q, k = torch.zeros(1, heads, queries, 64, dtype=HALF, device="cuda"), torch.zeros(1, 1, keys, 64, dtype=HALF, device="cuda")
    v = torch.full_like(k, -1.0)
    q[..., 0], k[0, 0, 0, 0], v[0, 0, 0] = 1.0, 13.0, 1.0
    apart = math.log(2.0 ** 24 / below)
    bias = torch.zeros(heads, queries + keys - 1, device="cuda")
    others = (keys - 1) * math.exp(-13.0 * (scale := torch.tensor(apart / 13.0).item()))
    want = (1 - others) / (1 + others)
    for given in (None, bias):
        with torch.no_grad():
            y = ops.op_attention(q, k, v, given, scale=scale).double()
        # the result's rounding, and the exponents' in 32 bits
        off = 2.0 ** -11 * abs(want) + 2 * keys * 2.0 ** -32 + 2.0 ** -17
        assert (y - want).abs().max() <= off, (float((y - want).abs().max()), off)
