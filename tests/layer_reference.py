"""What tests/test_gpu_checkpoint_*.py compare with: the layers' formulas in 64 bits, and how far 32-bit sums may be off them."""
import math

import torch

GROUP = 256
U = 2.0 ** -24          # half a step of float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """The step of the smallest values, which no relative bound covers."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def gamma(n):
    """n additions (and a few operations around them) in float32, each off by at most half a step."""
    return (n + 16) * U


def codes_of(x):
    """Codes, scale, min of the checkpoint of x [rows, cols] by the format's definition, for each group on its own."""
    x = x.float()
    codes, scales, mins = [], [], []
    for first in range(0, x.shape[1], GROUP):
        part = x[:, first:first + GROUP]
        mn, mx = part.amin(1, keepdim=True), part.amax(1, keepdim=True)
        scale = (255.0 / ((mx - mn).double() + 2e-6)).float()
        # product and sum are rounded together: 64 bits hold both exactly but for the last bits of the sum
        level = ((part - mn).double() * scale.double() + 0.5).float() - 0.5
        codes.append(level.clamp(0, 255).round())
        scales.append(scale)
        mins.append(mn)
    return torch.cat(codes, 1).to(torch.uint8), torch.cat(scales, 1), torch.cat(mins, 1)


def spread(stat, cols):
    """A per-group [rows, groups] tensor for every column."""
    return stat.repeat_interleave(GROUP, 1)[:, :cols]


def values_of(checkpoint_codes, scale, mn, cols):
    """What codes stand for, in 64 bits, and by how much float32 may miss it: the reciprocal, the product and the sum."""
    c = checkpoint_codes.view(torch.uint8)[:, :cols].double()
    s, m = spread(scale, cols).double(), spread(mn, cols).double()
    v = c / s + m
    return v, 2 * U * (c / s) + 2 * U * v.abs()


def activation(z, kind):
    """act(z), act'(z) in 64 bits."""
    if kind is None:
        return z, torch.ones_like(z)
    if kind == "gelu":
        phi = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if kind == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        t = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return z * s, s * (1 + z * (1 - s))


# act' and act'' of all three stay below these; the kernels' exponentials and error functions are within this of act' (absolute; relative to
# |z| + 1 for act), whatever the type
MAX_SLOPE = 1.13
FUNCTION = 2e-6


def close(got, want, bound, name):
    """Every element within its bound (float64 tensors)."""
    off = (got.double() - want).abs() - bound
    bad = ~(off <= 0)
    assert not bad.any(), "%s: %d of %d outside, worst %.3g over a bound of %.3g (want %.6g, got %.6g)" % (
        name, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bound.expand_as(off)[bad][off[bad].argmax()]),
        float(want[bad][off[bad].argmax()]), float(got.double()[bad][off[bad].argmax()]))
