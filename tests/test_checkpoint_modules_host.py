"""How a model's layers come to run on 8-bit checkpoints and stop to, as far as it goes without a GPU."""
import copy
import io
import pickle

import pytest
import torch
import torch.nn as nn

from gact import layers
from gact.conf import config
from gact.controller import Controller
from gact.cpp_extension import _abi


@pytest.fixture(autouse=True)
def _restore_config():
    saved = copy.copy(config.__dict__)
    yield
    config.__dict__.update(saved)


def a_model():
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(6, 8), nn.GELU(), nn.LayerNorm(8), nn.Linear(8, 3, bias=False))


def test_copies_of_attached_layers_are_torchs_own():
    """An average of the model's weights, say, whose layers nobody would take back."""
    model, x = a_model(), torch.randn(5, 6)
    kinds, want = [type(m) for m in model], model(x)
    model[0].extra = [1, 2]
    hooked = model[2].register_forward_hook(lambda m, a, y: y + 1)
    changed = layers.attach(model)
    held = io.BytesIO()
    torch.save(model[0], held)
    held.seek(0)
    average = torch.optim.swa_utils.AveragedModel(model)
    copies = [copy.deepcopy(model[0]), copy.copy(model[0]), pickle.loads(pickle.dumps(model[0])), torch.load(held, weights_only=False),
              average.module[0]]
    assert all(type(m) is nn.Linear and m.extra == [1, 2] for m in copies)
    assert [type(m) for m in average.module] == kinds and [type(m) for m in copy.deepcopy(model)] == kinds
    assert all(torch.equal(m(x), model[0](x)) for m in copies)
    twin = copy.deepcopy(model[2])
    assert torch.equal(twin(want.new_ones(2, 8)), model[2](want.new_ones(2, 8)))       # its hooks too
    assert type(model[0]) is layers.CheckpointedLinear and type(model[2]) is layers.CheckpointedLayerNorm
    layers.detach(changed)
    hooked.remove()
    assert [type(m) for m in model] == kinds and torch.equal(model(x), want)


def test_copies_of_layers_that_were_made_so_stay_so():
    own = layers.CheckpointedLinear(6, 8)
    assert layers.attach(own) == []
    for m in (copy.deepcopy(own), copy.copy(own), pickle.loads(pickle.dumps(own))):
        assert type(m) is layers.CheckpointedLinear and torch.equal(m.weight, own.weight)


def test_layers_stay_attached_until_the_last_controller_leaves():
    config.checkpoint_layers, config.auto_prec = True, False
    model = a_model()
    kinds, swapped = [type(m) for m in model], [layers.CheckpointedLinear, nn.GELU, layers.CheckpointedLayerNorm, layers.CheckpointedLinear]
    whole, part = Controller(model), Controller(model[0])
    for order in ((whole, part), (part, whole)):
        for c in (whole, part):
            c.install_hook()
        assert [type(m) for m in model] == swapped
        order[0].uninstall_hook()
        assert [type(m) for m in model] == (swapped if order[0] is part else swapped[:1] + kinds[1:])
        order[1].uninstall_hook()
        assert [type(m) for m in model] == kinds
    whole.install_hook()
    own = layers.CheckpointedLinear(8, 8)
    model.append(own)                       # was made so, and stays so
    part.install_hook()
    whole.uninstall_hook()
    whole.uninstall_hook()                  # gone already
    assert [type(m) for m in model] == swapped[:1] + kinds[1:] + [layers.CheckpointedLinear]
    part.uninstall_hook()
    assert [type(m) for m in model] == kinds + [layers.CheckpointedLinear] and not len(layers._held)


def test_library_refuses_products_of_codes_whose_rows_are_too_far_apart():
    """Past 32 bits of offset within a step: codes would be read from other rows."""
    L = _abi.lib()
    for ldc in ((1 << 20) + 16, 1 << 26, 1 << 34):
        assert L.gact_checkpoint_product(16, 8, 16, ldc, 16, 16, 2, 64, 8, 8, 16, None, None) == -2


def test_layers_that_were_parametrized_while_attached_are_detached():
    model, x = a_model(), torch.randn(5, 6)
    changed = layers.attach(model)
    for n in (0, 2):
        torch.nn.utils.parametrize.register_parametrization(model[n], "weight", nn.Softplus())
    twin, want = copy.deepcopy(model), model(x)
    layers.detach(changed)
    for m in (model, twin):
        assert not any(isinstance(layer, (layers.CheckpointedLinear, layers.CheckpointedLayerNorm)) for layer in m)
        assert torch.equal(m(x), want)
    torch.nn.utils.parametrize.remove_parametrizations(model[0], "weight")
    assert type(model[0]) is nn.Linear
