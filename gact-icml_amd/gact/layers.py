"""Layers that keep their input in 8 bits and train on it: checkpoints of rows, layer norm and linear layers.

The saved-tensor hooks of the Controller hand the backward pass a whole dequantized tensor.  These operators save their own input as
8-bit codes (a quarter or half of its bytes) and their backward kernels read the codes where they lie: no dequantized copy exists
at any time.  Rounding is to nearest, so a pass is repeatable and needs no seeds.

A checkpoint holds every row in groups of 256 columns, the last of them shorter, with a float scale and minimum each; its codes are those
of ``op_quantize(x.float(), 8, ..., rng_stream="deterministic")`` and, where 256 divides the columns, ``op_dequantize`` takes them.  As
there, a NaN among numbers becomes its group's minimum, and a group of NaN alone, or of a range beyond float's (an infinity's), becomes NaN: the
results of a row that is not finite are not finite, but a weight's gradient from a finite gradient of the result need not show a NaN of the input.

Arguments are float32, float16 or bfloat16 tensors on one GPU, of one type, with any strides; a layout that the kernels do not load is copied
first.  The work goes to the current stream.  Whatever cannot be taken raises a RuntimeError (a TypeError where no tensor
was given), before anything is launched.

The public names are in ``gact.ops``; nothing of this is in the reference, whose layers save through the hooks only.
"""
import collections
import weakref

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils._device import DeviceContext

from .cpp_extension import _abi

_ACTIVATIONS = {None: 0, "gelu": 1, "gelu_tanh": 2, "silu": 3}

# codes int8 [rows, stride] (stride: the columns rounded up to 16), scale and min float32 [rows, groups]; shape and dtype of the
# tensor it stands for
Checkpoint = collections.namedtuple("Checkpoint", "codes scale min shape dtype")


def op_checkpoint(input):
    """The 8-bit checkpoint of a float32, float16 or bfloat16 tensor [..., cols].  Codes are whole numbers: neither this nor op_restore has a
    derivative, and their results have no history."""
    codes, scale, mn = _abi.native().checkpoint(input)
    return Checkpoint(codes, scale, mn, input.shape, input.dtype)


def _parts(checkpoint):
    if not isinstance(checkpoint, Checkpoint):
        raise TypeError("a Checkpoint is expected")
    codes, scale, mn, shape, dtype = checkpoint
    return codes, scale, mn, tuple(shape), dtype


def op_restore(checkpoint):
    """The tensor a checkpoint stands for, in its shape and type."""
    return _abi.native().restore(*_parts(checkpoint))


def op_checkpoint_product(grad, checkpoint):
    """[outer, cols] = grad [..., outer] transposed times the checkpoint's values [..., cols], both as rows: the weight's gradient of a
    linear layer whose input the checkpoint holds.  The values enter the product in the checkpoint's type, as op_restore gives them.  It has no
    backward pass: going through the result of a gradient that has a history is an error."""
    return _abi.native().checkpoint_product(*_parts(checkpoint), grad)


def op_layer_norm(input, weight=None, bias=None, eps=1e-5):
    """Layer norm over the last dimension.  For the backward pass it keeps the 8-bit checkpoint of the input and each row's mean and
    1 / sqrt(var + eps); gradients are those of the checkpoint's values under that mean and deviation.  Under autocast it runs in
    float32, as torch's does."""
    return _abi.native().layer_norm(input, weight, bias, eps, torch.float32 if torch.is_autocast_enabled("cuda") else None)


def op_linear(input, weight, bias=None, activation=None, residual=None):
    """activation(input weight^T + bias) + residual in one kernel; activation None, "gelu", "gelu_tanh" or "silu".

    For the backward pass it keeps the 8-bit checkpoint of the input and, under an activation, of the value it is applied to; the
    gradients are those of the checkpoints' values; under an activation its gradient dz is rounded to the layer's type before dx and dW,
    as the matrix instructions take it (bias gradients add it up unrounded).  (relu is not among them: its derivative jumps at zero, where
    8 bits do not hold the sign.)  Under autocast it runs in autocast's type; the weight that it saves is the one it was given, which the backward pass rounds
    again."""
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise RuntimeError("unknown activation %r (expected one of %s)" % (activation, sorted(k for k in _ACTIVATIONS if k)))
    autocast = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None
    return _abi.native().linear(input, weight, bias, act, residual, autocast)


# ---- modules ----
def _overridden(tensors):
    """Whether a tensor's __torch_function__ or a mode's wants to see torch's call.  A default device is such a mode, too, and looks at
    calls that make tensors only."""
    return torch.overrides.has_torch_function(tensors) and not (
        all(type(t) in (torch.Tensor, nn.Parameter) for t in tensors)
        and all(isinstance(m, DeviceContext) for m in torch.overrides._get_current_function_mode_stack()))


def _taken(input, weight, bias, linear):
    """Whether the operator takes this call of a module: anything else goes to torch's own."""
    if not (isinstance(input, torch.Tensor) and input.is_cuda):
        return False
    return (not _overridden(tuple(t for t in (input, weight, bias) if t is not None))
            and _abi.native().takes(input, weight, bias, linear, torch.is_autocast_enabled("cuda")))


_attached = weakref.WeakSet()


class _Swapped:
    """Copies and pickles of a module that runs on an operator because it is attached are torch's own modules: nothing would ever detach them
    (a running average of the model, say), and they load where this package is not there.  A module that was made so stays so."""

    def __reduce_ex__(self, protocol):
        made = super().__reduce_ex__(protocol)
        return (object.__new__, (self._own,)) + made[2:] if self in _attached else made


class CheckpointedLinear(_Swapped, nn.Linear):
    """nn.Linear on op_linear."""
    _own = nn.Linear

    def forward(self, input):
        weight, bias = self.weight, self.bias       # once: either may be computed each time it is asked for
        if _taken(input, weight, bias, True):
            return op_linear(input, weight, bias)
        return F.linear(input, weight, bias)


class CheckpointedLayerNorm(_Swapped, nn.LayerNorm):
    """nn.LayerNorm over the last dimension on op_layer_norm."""
    _own = nn.LayerNorm

    def forward(self, input):
        weight, bias = self.weight, self.bias
        if len(self.normalized_shape) == 1 and _taken(input, weight, bias, False) and input.shape[-1] == self.normalized_shape[0]:
            return op_layer_norm(input, weight, bias, self.eps)
        return F.layer_norm(input, self.normalized_shape, weight, bias, self.eps)


_CHECKPOINTED = {nn.Linear: CheckpointedLinear, nn.LayerNorm: CheckpointedLayerNorm}


def attach(model):
    """The model's linear layers and layer norms (of exactly these classes) run on the operators from now on; returns them for detach."""
    changed = [m for m in model.modules() if type(m) in _CHECKPOINTED]
    for m in changed:
        m.__class__ = _CHECKPOINTED[type(m)]      # the module's parameters and hooks stay as they are
    _attached.update(changed)
    return changed


def detach(changed):
    """What attach returned, as torch's own again."""
    for m in changed:
        _attached.discard(m)
        for own, checkpointed in _CHECKPOINTED.items():
            if type(m) is checkpointed:
                m.__class__ = own
            elif type(m).__bases__ == (checkpointed,) and torch.nn.utils.parametrize.is_parametrized(m):
                type(m).__bases__ = (own,)      # parametrized meanwhile: the class is the module's and its copies' own


# attached module -> how many hold it
_held = weakref.WeakKeyDictionary()


def hold(model):
    """attach for one of several that may want the same layers; returns what is to be given to release.  Layers that were attached by `attach`
    itself, and modules that were made as Checkpointed ones, are not theirs."""
    modules = attach(model) + [m for m in model.modules() if m in _held]
    for m in modules:
        _held[m] = _held.get(m, 0) + 1
    return modules


def release(modules):
    """The layers are torch's own again once the last one that held them lets go."""
    for m in modules:
        _held[m] -= 1
        if _held[m] == 0:
            del _held[m]
            detach([m])
