"""The layers on 8-bit checkpoints as far as they go without a GPU: what the library refuses before it touches the GPU, what the
operators refuse, and how the Controller swaps a model's layers in and out."""
import copy
import io

import pytest
import torch
import torch.nn as nn

from gact import layers, ops
from gact.conf import config
from gact.controller import Controller
from gact.cpp_extension import _abi

EINVAL, EALIGN = -1, -2


@pytest.fixture(autouse=True)
def _restore_config():
    saved = copy.copy(config.__dict__)
    yield
    config.__dict__.update(saved)


def test_library_refuses_before_it_touches_the_gpu():
    L = _abi.lib()
    # x, dtype, rows, cols, ldx, codes, ldc, scale, min, stream
    assert L.gact_checkpoint(16, 3, 4, 8, 8, 16, 16, 16, 16, None) == EINVAL                   # type
    assert L.gact_checkpoint(16, 0, -1, 8, 8, 16, 16, 16, 16, None) == EINVAL
    assert L.gact_checkpoint(16, 0, 4, 0, 8, 16, 16, 16, 16, None) == EINVAL                   # no columns
    assert L.gact_checkpoint(16, 0, 4, 262145, 262145, 16, 262160, 16, 16, None) == EINVAL     # too many
    assert L.gact_checkpoint(16, 0, 4, 8, 7, 16, 16, 16, 16, None) == EINVAL                   # rows overlap
    assert L.gact_checkpoint(16, 0, 4, 8, 8, None, 16, 16, 16, None) == EINVAL
    assert L.gact_checkpoint(16, 0, 4, 8, 8, 16, 8, 16, 16, None) == EALIGN                    # codes' stride
    assert L.gact_checkpoint(16, 0, 4, 17, 17, 16, 16, 16, 16, None) == EALIGN                 # shorter than a row
    assert L.gact_checkpoint(16, 0, 0, 8, 8, None, 16, None, None, None) == 0                  # nothing to do
    assert L.gact_restore(16, 16, 16, 16, 0, 4, 8, 8, None) == EALIGN                          # out
    assert L.gact_pad_rows(16, 0, 4, 9, 9, 16, 8, None) == EALIGN and L.gact_pad_rows(16, 0, 4, 9, 9, 16, 12, None) == EALIGN
    norm = lambda cols, codes, ldc, scale: L.gact_norm_forward(16, cols, None, None, 0, 4, cols, 1e-5, 16, codes, ldc, scale, scale, scale, None)  # noqa: E731
    assert norm(16385, None, 0, None) == EINVAL and norm(8, 16, 16, None) == EINVAL and norm(8, 16, 24, 16) == EALIGN
    assert L.gact_norm_backward(16, 8, None, 16, 16, 16, 16, 16, 0, 0, 8, 16, None, None, None, None) == EINVAL    # no rows
    assert L.gact_norm_backward(16, 8, None, 16, 16, 16, 16, 16, 0, 4, 8, 16, 16, None, None, None) == EINVAL      # sums without workspace
    linear = lambda ldx=8, x=16, act=0, codes=None, rows=100, inner=8, ws=None: L.gact_linear(  # noqa: E731
        x, ldx, 16, 8, None, None, 0, act, 0, rows, inner, 8, 16, codes, 16, 16, 16, ws, None)
    assert linear(act=4) == EINVAL and linear(rows=-1) == EINVAL and linear(inner=0) == EINVAL
    assert linear(codes=16) == EINVAL                                                            # codes without an activation
    assert linear(x=8) == EALIGN and linear(ldx=9) == EALIGN and linear(ldx=4, inner=8) == EINVAL
    assert linear(ldx=4, rows=9) == EINVAL and linear(ldx=-8, rows=9) == EINVAL                  # rows over one another
    assert linear(act=1, codes=8) == EALIGN and linear(act=1, codes=16) == EALIGN and linear(act=1, codes=16, ws=8) == EALIGN   # workspace
    assert L.gact_linear(16, 1 << 21, 16, 8, None, None, 0, 0, 0, 100, 8, 8, 16, None, 0, None, None, None, None) == EALIGN   # beyond a tile's window
    act = lambda codes, which, dz, lddz, db, ws: L.gact_activation_backward(16, 9, codes, 16, 16, 16, which, 0, 4, 9, dz, lddz, db, ws, None)  # noqa: E731
    assert act(None, 1, 16, 16, None, None) == EINVAL and act(16, 1, None, 16, None, None) == EINVAL
    assert act(16, 1, 16, 16, 16, None) == EINVAL and act(16, 1, 16, 12, None, None) == EALIGN and act(16, 1, 16, 24, None, None) == EALIGN
    assert L.gact_product(16, 9, 16, 8, 0, 4, 9, 8, 16, None, None) == EALIGN                  # a's rows are no whole pieces
    assert L.gact_product(16, 8, 16, 8, 0, 4, 9, 8, 16, None, None) == EALIGN                  # and have no room for the last one
    assert L.gact_checkpoint_product(16, 8, 16, 16, 16, 16, 0, 0, 8, 8, 16, None, None) == EINVAL
    # deep and narrow: cut along the depth, into partial sums that need room
    assert L.gact_product_workspace_bytes(2, 128, 128, 1 << 16) > 0
    assert L.gact_product(16, 1 << 16, 16, 128, 2, 128, 1 << 16, 128, 16, None, None) == EALIGN


def test_workspaces_are_sized():
    L = _abi.lib()
    assert L.gact_norm_workspace_bytes(0, 8) == 0 and L.gact_norm_workspace_bytes(1, 96) == 2 * 96 * 4
    for rows in (1, 7, 1000, 10 ** 6):
        for cols in (1, 96, 1024, 5000, 16384):
            assert L.gact_norm_workspace_bytes(rows, cols) % (2 * cols * 4) == 0
            assert 0 < L.gact_norm_workspace_bytes(rows, cols) <= 512 * 2 * cols * 4
            assert 0 < L.gact_activation_workspace_bytes(rows, cols) <= 65535 * cols * 4
    # a product whose tiles fill the card needs none; otherwise whole partial results, at most 64
    assert L.gact_product_workspace_bytes(2, 8192, 8192, 4096) == 0
    for rows, cols, depth in ((1, 1, 1), (4096, 1024, 16384), (64, 64, 10 ** 6), (1285, 771, 3001)):
        size, one = L.gact_product_workspace_bytes(1, rows, cols, depth), rows * -(-cols // 4) * 16
        assert size % one == 0 and size <= 64 * one


def test_operators_refuse_what_is_not_on_the_gpu():
    x = torch.zeros(4, 8)
    for call in (lambda: ops.op_checkpoint(x), lambda: ops.op_layer_norm(x), lambda: ops.op_linear(x, x),
                 lambda: ops.op_linear(x, x, None, "gelu", x)):
        with pytest.raises(RuntimeError, match="data must be a CUDA tensor!"):
            call()
    for call in (lambda: ops.op_checkpoint([1.0]), lambda: ops.op_layer_norm(None), lambda: ops.op_linear(3, x)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(RuntimeError, match="unknown activation 'relu'"):
        ops.op_linear(x, x, None, "relu")
    with pytest.raises(TypeError):
        ops.op_restore((x, x, x))
    with pytest.raises(RuntimeError, match="do not belong"):
        ops.op_restore(ops.Checkpoint(torch.zeros(4, 16, dtype=torch.int8), x, x, torch.Size((4, 8)), torch.float32))
    with pytest.raises(RuntimeError, match="shape or type"):
        ops.op_restore(ops.Checkpoint(torch.zeros(4, 16, dtype=torch.int8), x, x, torch.Size((4, 8)), torch.int32))


class Scaled(nn.Linear):
    def forward(self, input):
        return 2 * super().forward(input)


def a_model():
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(6, 8), nn.GELU(), nn.LayerNorm(8), Scaled(8, 8), nn.LayerNorm((2, 8)), nn.Linear(8, 3, bias=False))


def test_layers_are_swapped_in_place_and_back():
    model, x = a_model(), torch.randn(5, 2, 6)
    want, kinds, weights = model(x), [type(m) for m in model], [id(p) for p in model.parameters()]
    changed = layers.attach(model)
    assert [type(m) for m in model] == [layers.CheckpointedLinear, nn.GELU, layers.CheckpointedLayerNorm, Scaled, layers.CheckpointedLayerNorm,
                                        layers.CheckpointedLinear]
    assert torch.equal(model(x), want)              # not on the GPU: torch's own
    assert layers.attach(model) == []               # nothing left to change
    twin = copy.deepcopy(model)
    twin[0].weight.data.zero_()
    assert model[0].weight.abs().sum() > 0 and twin[0](x).std(0).abs().sum() == 0       # a copy runs on its own weights
    held = io.BytesIO()
    torch.save(model, held)
    held.seek(0)
    assert torch.equal(torch.load(held, weights_only=False)(x), want)
    layers.detach(changed)
    assert [type(m) for m in model] == kinds and [id(p) for p in model.parameters()] == weights and torch.equal(model(x), want)


def test_controller_swaps_layers_only_where_it_is_asked_to():
    config.auto_prec = False
    model = a_model()
    kinds = [type(m) for m in model]
    with Controller(model):
        assert [type(m) for m in model] == kinds
    config.checkpoint_layers = True
    with Controller(model):
        assert type(model[0]) is layers.CheckpointedLinear and type(model[3]) is Scaled
    assert [type(m) for m in model] == kinds
    config.compress_activation = False              # level L0
    with Controller(model):
        assert [type(m) for m in model] == kinds
