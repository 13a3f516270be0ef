"""The row-wise operators under torch's transforms: an input with a forward-mode tangent is
refused, since the operators have no such derivative, and so is every tracer, which would record
the result's allocation alone. Without a GPU the C entries are stood in for; the same calls run
on the device below."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from src import ops
from src.ops import _lib, q4, rowwise


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
    monkeypatch.setattr(q4, "rows_of", rowwise.rows_of)
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


def _traces(device, call):
    for leaf in (False, True):
        x = torch.ones(4, 8, device=device, requires_grad=leaf)
        for tracer in (lambda: torch.jit.trace(call, (x,), check_trace=False),
                       lambda: make_fx(call)(x), lambda: make_fx(call, pre_dispatch=True)(x),
                       lambda: make_fx(call, tracing_mode="fake")(x),
                       lambda: torch.func.functionalize(call)(x)):
            with pytest.raises((RuntimeError, ValueError)):
                tracer()
        y = call(x)
        if leaf and y.requires_grad:           # the backward pass alone
            with pytest.raises(RuntimeError, match="traced"):
                make_fx(lambda g: torch.autograd.grad(y, x, g, retain_graph=True)[0])(y.detach())
        with FlopCounterMode(display=False):   # a mode that records no graph is none of this
            assert call(x).shape == y.shape


def _table(device):
    return ops.Q4Table(torch.zeros(3, 16, dtype=torch.uint8, device=device),
                       torch.ones(3, 1, device=device).bfloat16(), 8)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("call", [*CALLS, "q4_matmul", "quantize_q4"])
def test_tracing_is_refused(stand_in, call):
    table = _table(stand_in)
    _traces(stand_in, {"q4_matmul": lambda x: ops.q4_matmul(x, table),
                       "quantize_q4": lambda x: ops.quantize_q4(x).scale}.get(call)
            or CALLS[call])


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("call", [*CALLS, "q4_matmul", "quantize_q4", "dequantize"])
def test_tracing_is_refused_on_the_device(cuda, call):
    table = _table(cuda)
    _traces(cuda, {"q4_matmul": lambda x: ops.q4_matmul(x, table),
                   "quantize_q4": lambda x: ops.quantize_q4(x).scale,
                   "dequantize": lambda x: table.dequantize() + x.detach()[:3]}.get(call) or CALLS[call])


def test_row0_past_64_bits_is_refused(stand_in):
    """A C entry would see it modulo 2^64: another row's draws. The bound leaves room for the
    rows behind it."""
    x = torch.ones(4, 8)
    for row0 in (2 ** 62 + 1, 2 ** 63, 2 ** 64, 2 ** 64 + 5):
        for call in (lambda: ops.dropout(x, 0.1, 1, row0=row0),
                     lambda: ops.dropout_add_layer_norm(x, x, None, None, 0.1, 1, row0=row0)):
            with pytest.raises(ValueError, match="row0"):
                call()
    assert ops.dropout(x, 0.1, 1, row0=2 ** 62).shape == (4, 8)
    L, a = _lib.lib(), x.data_ptr()
    assert L.gnnrec_dropout_forward(0, 4, 8, a, 8, a, 8, 0.1, 1, None, 0, 2 ** 62 + 1, 1.0,
                                    None) == -1
    assert "row0" in L.gnnrec_last_error().decode()


@pytest.mark.parametrize("call", CALLS)
def test_export_is_refused(stand_in, call):
    class Module(torch.nn.Module):
        def forward(self, x):
            return CALLS[call](x)

    with pytest.raises(RuntimeError):
        torch.export.export(Module(), (torch.ones(4, 8),), strict=False)


@pytest.mark.gpu
@pytest.mark.parametrize("call", [*CALLS, "q4_matmul"])
def test_compiled_functions_run_the_operators(cuda, call):
    """A call runs between the compiled parts, for other sizes and in the backward pass too."""
    table = _table(cuda)
    op = CALLS.get(call) or (lambda x: ops.q4_matmul(x.detach(), table))

    def both(x):
        return op(x * 2.0) + 1.0

    compiled = torch.compile(both, backend="eager")
    for rows in (4, 9):
        x = torch.randn(rows, 8, device=cuda, requires_grad=True)
        y, z = both(x), compiled(x)
        assert torch.equal(y, z)
        if y.requires_grad:
            g = torch.randn_like(y)
            assert torch.equal(torch.autograd.grad(y, x, g)[0], torch.autograd.grad(z, x, g)[0])
