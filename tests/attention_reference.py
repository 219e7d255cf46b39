"""What tests/test_gpu_attention*.py compare with: attention and its gradients in 64 bits, and how far the kernels' arithmetic may be off them, element by
element.

The kernels multiply in the tensors' type with sums in 32 bits, make exponentials of base 2 with the hardware's instruction (off by a unit in the last
place), and round probabilities and ds to the type before they enter a product; everything else is in 32 bits.  h is half a step of the type, U of float32.
A probability of float16 below 2^-14 is off by up to 2^-25 whatever it is; a row's largest unnormalised probability is 1 at least, so the same holds of the
normalised ones, and ds, which is not scaled, is off by that much itself."""
import math

import torch

from layer_reference import U, gamma, half_step, least

# the hardware's exponential gives zero where the result is below float's smallest normal number: a probability below 2^-126 is off by all of itself, and
# ds by that times do.v - do.o
FLUSHED = 2.0 ** -126


def attend(q, k, v, dy=None, bias=None, mask=None, causal=False, scale=None):
    """dict of (value, bound) pairs: y, and with dy also dq, dk, dv and, with a bias, dbias."""
    dtype = q.dtype
    h = half_step(dtype)
    small = 2.0 ** -25 if dtype is torch.float16 else FLUSHED
    q, k, v = (t.detach().double() for t in (q, k, v))
    (b, heads, m, w), (kv, n) = q.shape, k.shape[1:3]
    r = heads // kv
    scale = 1 / math.sqrt(w) if scale is None else scale
    K, V = k.repeat_interleave(r, 1), v.repeat_interleave(r, 1)
    if mask is not None:        # what is absent is not looked at
        there = mask[:, None, :, None]
        K, V = torch.where(there, K, 0.0), torch.where(there, V, 0.0)
    s = scale * (q @ K.mT)
    size = scale * (q.abs() @ K.abs().mT)
    i, j = torch.arange(m, device=q.device)[:, None], torch.arange(n, device=q.device)[None, :]
    seen = torch.ones(b, heads, m, n, dtype=torch.bool, device=q.device)
    if bias is not None:
        add = bias.detach().double()[:, (j - i + m - 1)]
        seen &= add > -1e30
        add = torch.where(add > -1e30, add, 0.0)
        s, size = s + add, size + add.abs()
    if mask is not None:
        seen &= mask[:, None, None, :]
    if causal:
        seen &= j <= i + n - m
    some = seen.any(3, keepdim=True)
    s = s.masked_fill(~seen, -math.inf)
    most = torch.where(some, s.amax(3, keepdim=True) if n else 0.0, 0.0)
    p = torch.exp(s - most)
    total = p.sum(3, keepdim=True)
    p = p / torch.where(some, total, 1.0)
    lse = most + torch.log(torch.where(some, total, 1.0))
    # the score's error: its sum, the factors' roundings, the exponent's
    e = torch.where(seen, (gamma(w) + 8 * U) * size + 4 * U * most.abs() + 4 * U, 0.0)
    worst = e.amax(3, keepdim=True) if n else torch.zeros_like(most)
    y, size_y = p @ V, p @ V.abs()
    off_y = (2 * worst + h + gamma(n) + 16 * U) * size_y + small * (seen.double() @ V.abs()) + h * y.abs() + least(dtype)
    out = {"y": (y, off_y)}
    if dy is None:
        return out
    dy = dy.detach().double()
    rel = e + worst + gamma(n) + 8 * U * lse.abs() + 16 * U         # of a probability that is computed again
    dp, size_dp = dy @ V.mT, dy.abs() @ V.abs().mT
    delta = (dy * y).sum(3, keepdim=True)
    off_delta = (dy.abs() * off_y).sum(3, keepdim=True) + gamma(w) * (dy.abs() * (y.abs() + off_y)).sum(3, keepdim=True)
    ds = p * (dp - delta)
    off_ds = p * (rel * (dp - delta).abs() + gamma(w) * size_dp + off_delta + 4 * U * (dp.abs() + delta.abs())) + FLUSHED * (dp - delta).abs()
    in_product = off_ds + h * (ds.abs() + off_ds) + small
    in_product = torch.where(seen, in_product, 0.0)

    def shared(t):
        return t.view(b, kv, r, n, w).sum(2)

    dv = shared(p.mT @ dy)
    off_dv = shared(((rel + h) * p + torch.where(seen, small, 0.0)).mT @ dy.abs()) + gamma(m * r) * shared(p.mT @ dy.abs())
    dq = scale * (ds @ K)
    off_dq = scale * (in_product @ K.abs() + (gamma(n) + 4 * U) * (ds.abs() @ K.abs()))
    dk = scale * shared(ds.mT @ q)
    off_dk = scale * (shared(in_product.mT @ q.abs()) + (gamma(m * r) + 4 * U) * shared(ds.abs().mT @ q.abs()))
    for name, value, off in (("dq", dq, off_dq), ("dk", dk, off_dk), ("dv", dv, off_dv)):
        out[name] = value, off * (1 + h) + h * value.abs() + least(dtype)
    if bias is not None:
        at = (j - i + m - 1).expand(b, heads, m, n)

        def along(t):
            sums = torch.zeros(heads, m + n - 1, dtype=torch.float64, device=q.device)
            return sums.scatter_add_(1, at.transpose(0, 1).reshape(heads, -1), t.transpose(0, 1).reshape(heads, -1))

        out["dbias"] = along(ds), along(off_ds) + gamma(b * m) * along(ds.abs()) + least(torch.float32)
    return out
