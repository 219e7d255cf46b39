"""Attention that trains without its probabilities, and a relative position bias by buckets.

The probabilities are the largest tensor that a layer of a transformer saves.  ``op_attention`` saves its three inputs, its result (with a byte for each
16-bit value of what its rounding left out) and one float per query and head; its backward pass computes the probabilities again, a tile at a time, and neither they nor their gradient are ever in memory.  The
position bias is held as one value per head and distance, not per query and key, and so is its gradient.

Arguments are float32, float16 or bfloat16 tensors on one GPU, of one type, with any strides; a layout that the kernels do not load is copied first.  The
work goes to the current stream, sums are made in one order (a pass is repeatable), and whatever cannot be taken raises a RuntimeError (a TypeError
where no tensor was given), before anything is launched.

The public names are in ``gact.ops``; nothing of this is in the reference, whose layers save the probabilities through the hooks.
"""
import torch

from .cpp_extension import _abi


def op_attention(query, key, value, bias=None, mask=None, causal=False, scale=None):
    """softmax(scale query key^T + bias) value for query [batch, heads, queries, width] and key and value [batch, key heads, keys, width]; every key
    head serves heads / key heads neighbouring heads.  width 1 to 128; scale 1 / sqrt(width) where none is given.

    bias: float32 [heads, queries + keys - 1], added at j - i + queries - 1 (op_position_bias makes one); values of -1e30 or less hide the key.
    mask: bool [batch, keys], which keys are there.  What absent keys and values hold does not matter.
    causal: query i sees the keys up to i + keys - queries: the last query sees all of them.  A NaN of a key that is hidden in this way may show.
    A query that nothing is left for gets zeros, and gives none of its gradient to anyone, NaN and infinity included.

    In 16-bit types the probabilities are rounded before they meet the values, and with a bias what that leaves out is added: the result is then off by little
    more than its own rounding, without a bias by a fifth (bfloat16) or a third (float16) more in norm.

    The result lies in memory as [batch, queries, heads, width], so that its transpose(1, 2) is a projection's contiguous input.  Under hooks for saved
    tensors (the Controller's) query, key and value, and a mask, are all that they get; the bias is held as it is, and the backward pass runs the forward
    pass again on what the hooks give back: the gradients are exactly those of these values.  Under autocast it runs in autocast's type, the bias in float32."""
    autocast = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None
    return _abi.native().attention(query, key, value, bias, mask, causal, scale, autocast)


def op_position_bias(table, queries, keys, bidirectional=True, max_distance=128):
    """A learned bias by distance, [heads, queries + keys - 1] float32, out of table [buckets, heads]: the bias of distance d = key - query is at
    d + keys - 1, for queries that are the last ones of the keys (as in op_attention).

    bidirectional: half of the buckets are for keys behind the query, half for itself and those before it; otherwise all are for keys before it, and the
    keys behind share the first one with the query itself.  Of one direction's buckets the first half hold a distance each, the others
    reach up to max_distance in equal steps of its logarithm, and the last one has everything further off."""
    return _abi.native().position_bias(table, queries, keys, bidirectional, max_distance)
