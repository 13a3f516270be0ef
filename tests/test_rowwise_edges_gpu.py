"""Calls of the row-wise operators at the edges of what they document, on the GPU."""
import pytest
import torch

import rowwise_ref as R
from src import ops

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _randn(*shape, dtype=F32, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) + shift).to(dtype).cuda()


@pytest.mark.parametrize("p,slope,with_res", [(0.0, 1.0, True), (0.3, 0.2, True),
                                              (0.3, 1.0, False), (1.0, 0.2, False)])
@pytest.mark.parametrize("d", [5, 64, 300])
def test_gradients_of_h_alone_do_not_pass_the_norm(cuda, d, p, slope, with_res):
    """Rows that have no norm (a NaN, an infinity, a constant row without eps) leave the
    gradients that come through h alone as they are: dx = dh s act'(x), dres = dh, dw = db = 0."""
    x, res = _randn(9, d), _randn(9, d, seed=1)
    x[1, 2], x[3, 0], x[5] = float("nan"), float("inf"), 2.0
    res[5], res[7, 1] = 1.0, float("-inf")
    w, b, dh = _randn(d, seed=2), _randn(d, seed=3), _randn(9, d, seed=4)
    leaves = [t.requires_grad_() for t in ((x, res, w, b) if with_res else (x, w, b))]
    _, h = ops.dropout_add_layer_norm(x, res if with_res else None, w, b, p, 5,
                                      negative_slope=slope, eps=0.0)
    got = torch.autograd.grad(h, leaves, dh)
    f = R.drop_factor(9, d, p, 5) * torch.where(x.detach().cpu() > 0, 1.0, slope)
    want = dh.cpu().double() * f
    R.assert_close(got[0], want, 5 * R.U * want.abs(), "dx")
    if with_res:
        assert torch.equal(got[1], dh)
    assert not got[-2].any() and not got[-1].any()
    # an expanded gradient (a sum's)
    _, h = ops.dropout_add_layer_norm(x, res if with_res else None, w, b, p, 5,
                                      negative_slope=slope, eps=0.0)
    R.assert_close(torch.autograd.grad(h.sum(), x)[0], f, 5 * R.U * f)
