"""NGCF's counter-based dropout and layer norm beside what its plain form takes."""
import pytest
import torch

from test_row_operator_paths import _graph, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_norm_under_autocast(cuda, dtype):
    """The Linear layers' sum is in half precision then, the residual in fp32: the sum and the
    norm are in fp32, as the next hop needs its table. Against the fp32 forward, by the norm of
    the whole: a product's two roundings (0.6 half steps each in the mean square) and three of
    the results come to 1.3 half steps of z, times at most 4 of a norm's scale, for each of three
    layers: 16 half steps."""
    g, _ = _graph()
    g = g.to(cuda)
    m = _model(layer_norm=True).to(cuda).eval()
    out, grad = {}, {}
    for on in (False, True):
        with torch.autocast("cuda", dtype=dtype, enabled=on):
            x = torch.cat(m(g))
        assert x.dtype == torch.float32
        x.sum().backward()
        out[on] = x.detach()
        grad[on] = m.user_embedding.weight.grad
        m.zero_grad()
    assert torch.isfinite(grad[True]).all()
    step = torch.finfo(dtype).eps / 2
    assert (out[True] - out[False]).norm() < 16 * step * out[False].norm()
    m.train()
    with torch.autocast("cuda", dtype=dtype):
        x = torch.cat(m(g))
    x.sum().backward()
    assert x.dtype == torch.float32 and torch.isfinite(m.user_embedding.weight.grad).all()


@pytest.mark.parametrize("kw", [dict(counter_dropout=True), dict(layer_norm=True)])
def test_masks_are_drawn_where_a_layer_drops(cuda, kw):
    """A layer decides by its own mode and rate whether it drops: one that was switched after the
    model was built, or alone (dropout at inference), draws like torch's dropout does."""
    g, _ = _graph()
    g = g.to(cuda)
    m = _model(**kw).to(cuda).eval()
    still = torch.cat(m(g)).detach()
    assert torch.equal(still, torch.cat(m(g)))
    m.layers[1].train()
    torch.manual_seed(1)
    one = torch.cat(m(g)).detach()
    assert torch.equal(one[:, :128], still[:, :128]) and not torch.equal(one, still)
    torch.manual_seed(1)
    with torch.no_grad():
        torch.testing.assert_close(torch.cat(m(g)), one, rtol=1e-4, atol=1e-5)
    m.eval()
    m.layers[1].dropout.train()                  # the dropout alone
    torch.manual_seed(1)
    assert torch.equal(torch.cat(m(g)), one)
    m.train()
    for layer in m.layers:
        layer.dropout.p = 0.0
    assert torch.equal(torch.cat(m(g)), torch.cat(m(g)))
    m.layers[0].dropout.p = 0.5
    m.dropout = 0.0
    assert not torch.equal(torch.cat(m(g)), torch.cat(m(g)))


def test_a_captured_step_needs_a_seed_on_the_device(cuda):
    """A seed drawn on the host would be every replay's."""
    g, _ = _graph()
    g = g.to(cuda)
    m = _model(counter_dropout=True).to(cuda).train()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        m(g)
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            with pytest.raises(RuntimeError, match="dropout_seed"):
                m(g)
            kept = torch.zeros(4, device=cuda).add_(1)      # the capture itself goes on
        m.eval()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                       # nothing is drawn: no seed needed
            out = torch.cat(m(g))
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, torch.cat(m(g)))
    del kept
