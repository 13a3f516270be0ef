"""The row-wise operators under torch's transforms: an input with a forward-mode tangent is
refused, since the operators have no such derivative. Without a GPU the C entries are stood in
for; the same calls run on the device below."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from src import ops
from src.ops import rowwise


@pytest.fixture
def stand_in(monkeypatch):
    """The operators on CPU tensors, their C entries replaced by ones that do nothing."""
    class Entries(dict):
        def get(self, name, default=None):
            return lambda *args: 0

    monkeypatch.setattr(rowwise, "_ENTRIES", Entries())
    monkeypatch.setattr(rowwise, "_current_device", lambda: None)
    monkeypatch.setattr(rowwise, "_raw_stream", lambda i: 0)
    monkeypatch.setattr(rowwise, "rows_of", lambda t, what: t.view(-1, t.shape[-1]))
    return torch.device("cpu")


CALLS = {
    "dropout": lambda x: ops.dropout(x, 0.1, 1),
    "layer_norm": lambda x: ops.layer_norm(x),
    "block": lambda x: ops.dropout_add_layer_norm(x, None, None, None, 0.1, 1)[0],
}


def _tangents(device, call):
    x = torch.ones(4, 8, device=device)
    for leaf in (False, True):
        for recording in (torch.enable_grad, torch.no_grad):
            with fwd.dual_level(), recording():
                dual = fwd.make_dual(x.clone().requires_grad_(leaf), torch.ones_like(x))
                with pytest.raises(NotImplementedError, match="jvp"):
                    call(dual)
    with fwd.dual_level():                     # inputs without a tangent are as ever
        assert call(x).shape == x.shape
        leaf = x.clone().requires_grad_()
        y = call(leaf)
        assert torch.autograd.grad(y, leaf, x, retain_graph=True)[0].shape == x.shape
        with pytest.raises(NotImplementedError, match="forward-mode"):     # a dual gradient
            torch.autograd.grad(y, leaf, fwd.make_dual(x, x))


@pytest.mark.parametrize("call", CALLS)
def test_tangents_are_refused(stand_in, call):
    _tangents(stand_in, CALLS[call])


def test_tangents_of_other_inputs_are_refused(stand_in):
    x, w = torch.ones(4, 8), torch.ones(8)
    with fwd.dual_level():
        dw, dr = fwd.make_dual(w, w), fwd.make_dual(x, x)
        for call in (lambda: ops.layer_norm(x, dw), lambda: ops.layer_norm(x, None, dw),
                     lambda: ops.dropout_add_layer_norm(x, dr, w, w, 0.1, 1)):
            with pytest.raises(NotImplementedError, match="jvp"):
                call()


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_tangents_are_refused_on_the_device(cuda, call):
    _tangents(cuda, CALLS[call])
