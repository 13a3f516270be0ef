"""NGCF layers and models made before their row-wise options, or by the caller."""
import copy

import pytest
import torch

from src.models import NGCF, NGCFGroupShuffle
from src.models.baselines.ngcf import NGCFLayer
from test_models import torch_adj
from test_row_operator_paths import _model


class OwnLayer(NGCFLayer):
    """A caller's layer with the arguments that a layer had."""

    def forward(self, x, adj_matrix, gas=None):
        n = torch.sparse.mm(adj_matrix, x)
        out = self.activation(self.W1(n) + self.W2(x * n))
        return gas(out) if gas is not None else out


@pytest.mark.parametrize("cls", [NGCF, NGCFGroupShuffle])
def test_layers_with_the_former_arguments(cls):
    m = _model(cls).eval()
    adj, _, _ = torch_adj()
    with torch.no_grad():
        want = torch.cat(m(adj))
        for k, layer in enumerate(m.layers):
            own = OwnLayer(layer.W1.in_features, layer.W1.out_features, 0.1)
            own.load_state_dict(layer.state_dict())
            m.layers[k] = own
        for mode in (False, True):
            assert torch.equal(torch.cat(m.train(mode)(adj)), want)


@pytest.mark.parametrize("cls", [NGCF, NGCFGroupShuffle])
def test_models_made_before_the_options(cls):
    """A model object that was saved whole has none of the options' attributes."""
    m = _model(cls).eval()
    adj, _, _ = torch_adj()
    state = copy.deepcopy(m.__dict__)
    state.pop("dropout_seed", None)
    for layer in state["_modules"]["layers"]:
        layer.__dict__.pop("counter_dropout")
        layer.__dict__.pop("norm", None)
        layer._modules.pop("norm", None)
    old = cls.__new__(cls)
    for k, layer in enumerate(state["_modules"]["layers"]):
        again = NGCFLayer.__new__(NGCFLayer)
        again.__setstate__(layer.__dict__)
        state["_modules"]["layers"][k] = again
    old.__setstate__(state)
    with torch.no_grad():
        assert torch.equal(torch.cat(old(adj)), torch.cat(m(adj)))
    torch.manual_seed(3)
    want = torch.cat(m.train()(adj))
    torch.manual_seed(3)
    assert torch.equal(torch.cat(old.train()(adj)), want)
    new = copy.deepcopy(_model(cls, layer_norm=True, counter_dropout=True))
    assert all(layer.norm is not None and layer.counter_dropout for layer in new.layers)
