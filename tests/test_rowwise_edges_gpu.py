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


def _room(gib):
    free, _ = torch.cuda.mem_get_info()
    if free < gib << 30:
        pytest.skip(f"needs {gib} GiB of device memory, {free >> 30} are free")


@pytest.mark.parametrize("what", ["dropout", "layer_norm", "quantize", "users"])
def test_more_threads_than_a_grid_dimension_takes(cuda, what):
    """Tables of more than 2^32 threads' work: narrow rows of one row's view, so that little
    memory is needed for them; the far rows are those of a small call."""
    torch.cuda.empty_cache()
    n = 2 ** 32 + 1000
    if what == "dropout":                        # a thread a row
        _room(40)
        x = _randn(1, 1, dtype=BF16, shift=2.0).expand(n, 1).requires_grad_()
        y = ops.dropout(x, 0.4, 7, negative_slope=0.2)
        dx, = torch.autograd.grad(y, x, x.detach())
        for r in (0, 2 ** 32 - 200, n - 300):
            part = x.detach()[:300].requires_grad_()
            z = ops.dropout(part, 0.4, 7, row0=r, negative_slope=0.2)
            dz, = torch.autograd.grad(z, part, part.detach())
            assert torch.equal(y[r:r + 300], z[:n - r]) and torch.equal(dx[r:r + 300], dz[:n - r])
    elif what == "layer_norm":                   # fp32: a lane a row, a workgroup 256 rows
        _room(40)
        x = _randn(1, 2).expand(n, 2)
        y = ops.layer_norm(x)
        for r in (0, 2 ** 32 - 200, n - 300):
            assert torch.equal(y[r:r + 300], ops.layer_norm(x[:300]))
    elif what == "quantize":                     # four threads a row
        _room(40)
        n = 2 ** 30 + 1000
        w = torch.tensor([[-3.0]], device=cuda).expand(n, 1)
        t = ops.quantize_q4(w)
        small = ops.quantize_q4(w[:300])
        scores = ops.q4_matmul(torch.ones(1, 1, device=cuda), t)
        values = t.dequantize()
        want = small.dequantize()
        for r in (0, 2 ** 30 - 200, n - 300):
            assert torch.equal(t.codes[r:r + 300], small.codes)
            assert torch.equal(t.scale[r:r + 300], small.scale)
            assert torch.equal(values[r:r + 300], want)
            assert torch.equal(scores[0, r:r + 300], want[:, 0])
    else:                                        # a thread eight values of a user's row
        _room(100)
        m, k = 65535, 8 * 65536 + 13
        x = _randn(1, k, dtype=BF16).expand(m, k)
        t = ops.quantize_q4(_randn(2, k, seed=1))
        got = ops.q4_matmul(x, t)
        assert torch.equal(got, ops.q4_matmul(x[:1], t).expand(m, 2))
    torch.cuda.empty_cache()
