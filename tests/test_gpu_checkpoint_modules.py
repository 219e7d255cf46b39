"""A model's layers on 8-bit checkpoints where torch's own would be called in other ways than a plain training step: autocast under the
Controller's hooks."""
import copy

import pytest
import torch
import torch.nn as nn

from gact import layers
from gact.conf import config
from gact.controller import Controller

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _restore_config():
    saved = copy.copy(config.__dict__)
    yield
    config.__dict__.update(saved)


def normal(*shape, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * len(shape))
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_autocast_under_the_hooks_keeps_the_weights_as_they_are(dtype):
    """The hooks compress what a layer saves, but for a model's parameters: none of these layers' tensors is theirs."""
    config.checkpoint_layers, config.auto_prec, config.bit = True, False, 2
    model = nn.Sequential(nn.Linear(64, 48), nn.LayerNorm(48), nn.Linear(48, 40)).cuda()
    x, dy = normal(130, 64).requires_grad_(), normal(130, 40, dtype=dtype, seed=1)
    leaves = [x] + list(model.parameters())

    def step():
        with torch.autocast("cuda", dtype=dtype):
            y = model(x)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))

    changed = layers.attach(model)
    want = step()
    layers.detach(changed)
    controller = Controller(model)
    with controller:
        got = step()
    assert controller.quantizer.tid == 0
    assert all(torch.equal(a, b) and a.dtype is b.dtype for a, b in zip(got, want))
    assert all(g.dtype is torch.float32 for g in got[1:])


def test_autocast_keeps_no_copy_of_the_weight():
    """And its gradients are those of the weight rounded beforehand."""
    x, w = normal(70, 264, dtype=torch.bfloat16).requires_grad_(), normal(520, 264, seed=1, scale=0.1).requires_grad_()
    dy, rounded = normal(70, 520, dtype=torch.bfloat16, seed=2), w.detach().bfloat16().requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layers.op_linear(x, w, None, "gelu")
    codes = 70 * (272 + 528) + 70 * (2 + 3) * 8
    assert torch.cuda.memory_allocated() - before <= y.numel() * 2 + codes + 7 * 512 < y.numel() * 2 + w.numel() * 2
    z = layers.op_linear(x, rounded, None, "gelu")
    assert torch.equal(y, z)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    want = torch.autograd.grad(z, [x, rounded], dy)
    assert torch.equal(dx, want[0]) and dw.dtype is torch.float32 and torch.equal(dw, want[1].float())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layers.op_linear(x, w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], dy)
    empty = torch.empty(0, 264, device="cuda", requires_grad=True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layers.op_linear(empty, w)
    dw, = torch.autograd.grad(y, [w], torch.empty_like(y))
    assert dw.dtype is torch.float32 and not dw.any()


def test_a_capture_beside_an_eager_graph_is_refused_under_autocast():
    """Whichever argument is the leaf: what the operator runs on is a copy of it, and its backward pass ends in the leaf."""
    x, w, b, r = normal(40, 32), normal(24, 32, seed=1), normal(24, seed=2), normal(40, 24, seed=3)
    half = normal(40, 32, dtype=torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for n in range(4):
            args = [t.clone().requires_grad_(k == n) for k, t in enumerate((x, w, b, r))]
            eager = layers.op_linear(args[0], args[1], args[2], None, args[3])
            with pytest.raises(RuntimeError, match="eager graph of one of its leaves"):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    layers.op_linear(args[0], args[1], args[2], None, args[3])
            torch.autograd.grad(eager, [args[n]], torch.ones_like(eager))
            del eager
        leaf = half.clone().requires_grad_()
        eager = layers.op_layer_norm(leaf)
        with pytest.raises(RuntimeError, match="eager graph of one of its leaves"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                layers.op_layer_norm(leaf)


def test_refusals_under_autocast():
    x, w = normal(8, 16), normal(4, 16, seed=1)
    with torch.autocast("cuda", dtype=torch.float16):
        for bad in (lambda: layers.op_linear(x, w.double()), lambda: layers.op_linear(x.double(), w), lambda: layers.op_linear(x, w, normal(4).int()),
                    lambda: layers.op_layer_norm(x.double())):
            with pytest.raises(RuntimeError, match="type of"):
                bad()
        with pytest.raises(RuntimeError, match="dimension of bias"):
            layers.op_linear(x, w, normal(5))
        with pytest.raises(RuntimeError, match="dimension of weight"):
            layers.op_layer_norm(x, normal(8))
        with pytest.raises(RuntimeError, match="residual"):
            layers.op_linear(x, w, None, None, normal(8, 5))
        with pytest.raises(RuntimeError, match="CUDA"):
            layers.op_linear(x, w.cpu())
