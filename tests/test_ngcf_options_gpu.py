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
