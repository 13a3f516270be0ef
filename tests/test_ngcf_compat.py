"""NGCF over layers of the caller's own."""
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
