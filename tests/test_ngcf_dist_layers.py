"""The sharded NGCF forward over layers that know nothing of the norm."""
from types import SimpleNamespace

import torch

from src.models import NGCF
from src.ops.distributed import DistributedGraph, ngcf_forward_dist
from test_distributed import cpu_ngcf_layer
from test_row_operator_paths import _graph, _model


def test_layers_without_a_norm_attribute():
    """Its own layer function reads a layer's two products and its activation only."""
    g, adj = _graph()
    m = _model(NGCF).eval()
    dg = DistributedGraph(g, 0, 1, "cpu")
    plain = SimpleNamespace(layers=[SimpleNamespace(W1=layer.W1, W2=layer.W2,
                                                    activation=layer.activation)
                                    for layer in m.layers])
    with torch.no_grad():
        x0 = dg.pad_table(m._initial_table())
        assert torch.equal(ngcf_forward_dist(dg, plain, x0, layer_fn=cpu_ngcf_layer),
                           ngcf_forward_dist(dg, m, x0, layer_fn=cpu_ngcf_layer))
