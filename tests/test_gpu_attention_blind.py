"""Queries that see nothing: their gradient is nobody's, whatever it holds."""
import math

import pytest
import torch

from gact import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + 7919 * sum(shape))
    return (torch.randn(*shape, generator=g) * scale).to(dtype).cuda()


# one kernel for short sequences, two for longer ones, splits of either side, shared key heads
@pytest.mark.parametrize("dtype", TYPES, ids=lambda t: str(t)[6:])
@pytest.mark.parametrize("shape", [(3, 2, 2, 64, 50, 64), (2, 4, 2, 33, 64, 32), (520, 2, 1, 40, 20, 128), (3, 2, 2, 130, 100, 64), (1, 4, 2, 700, 650, 128), (2, 2, 1, 300, 1100, 72),
                                   (64, 8, 8, 260, 256, 64), (2, 2, 2, 1, 500, 64)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", ["mask", "causal", "both", "bias"])
def test_gradients_of_queries_that_see_nothing(kind, shape, dtype):
    b, h, g, m, n, w = shape
    q, k, v, dy = normal(b, h, m, w, dtype=dtype), normal(b, g, n, w, dtype=dtype, seed=1), normal(b, g, n, w, dtype=dtype, seed=2), normal(b, h, m, w, dtype=dtype, seed=3)
    mask = bias = None
    causal = kind in ("causal", "both")
    i, j = torch.arange(m, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
    seen = torch.ones(b, h, m, n, dtype=torch.bool, device="cuda")
    if kind in ("mask", "both"):
        mask = torch.ones(b, n, dtype=torch.bool, device="cuda")
        mask[0] = False
        mask[1:, : n // 3] = False
        if b > 1:
            mask[-1, : n - 2] = False
        seen &= mask[:, None, None]
    if causal:
        seen &= j <= i + n - m
    if kind == "bias":
        bias = normal(h, m + n - 1, seed=4)
        bias[0, : m + n // 2] = -math.inf       # the first queries of the first head see some keys, the last ones none
        seen &= (bias > -1e30)[:, j - i + m - 1]
    blind = ~seen.any(3)
    leaves = [t.requires_grad_() for t in (q, k, v) + ((bias,) if bias is not None else ())]
    y = ops.op_attention(q, k, v, bias, mask, causal)
    assert not y[blind].any()
    clean = dy.clone()
    clean[blind] = 0
    want = torch.autograd.grad(y, leaves, clean, retain_graph=True)
    for bad in (math.nan, math.inf, -math.inf):
        dy[blind] = bad
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        for name, a, c in zip(("dq", "dk", "dv", "dbias"), got, want):
            assert torch.isfinite(a).all() and torch.equal(a, c), (name, bad)
