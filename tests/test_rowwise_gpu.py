"""Dropout, layer norm and the block between two hops on the GPU, against the plain 64-bit forms
of rowwise_ref.py within the bounds derived there."""
import pytest
import torch

import rowwise_ref as R
from src import ops
from src.ops import _lib
from src.ops.rowwise import launch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SEED = 0x1234567_89ABCDEF


def _randn(*shape, dtype=F32, seed=0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) + shift).to(dtype).cuda()


def _drop_bound(x, f, slope):
    """Bound of dropout(x): slope, scale and two products, each rounded."""
    v = R.leaky(x.double().cpu(), slope) * f
    return torch.where(f != 0, v, 0.0), 4 * R.U * v.abs()


# ---- dropout ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 8), (2, 9), (257, 64), (100, 321),
                                    (1, 5000), (40, 1000)])
@pytest.mark.parametrize("p,slope", [(0.1, 0.2), (0.5, 1.0)])
def test_dropout(cuda, dtype, rows, d, p, slope):
    x, dy = _randn(rows, d, dtype=dtype), _randn(rows, d, dtype=dtype, seed=1)
    x.requires_grad_()
    y = ops.dropout(x, p, SEED, site=3, negative_slope=slope)
    dx, = torch.autograd.grad(y, x, dy)
    f = R.drop_factor(rows, d, p, SEED, site=3)
    R.assert_close(y, *_drop_bound(x.detach(), f, slope), "y")
    want = dy.double().cpu() * torch.where(x.detach().cpu() > 0, 1.0, slope) * f
    R.assert_close(dx, want, 4 * R.U * want.abs(), "dx")


def test_dropout_borders(cuda):
    """p = 0 and 1, a p that rounds to either, and the largest that does not drop everything."""
    x = _randn(64, 33)
    for p in (0.0, 1e-6):
        assert torch.equal(ops.dropout(x, p, 1), x)
    for p in (1.0, 1 - 1e-6):
        x.requires_grad_()
        y = ops.dropout(x, p, 1, negative_slope=0.2)
        dx, = torch.autograd.grad(y.sum(), x)
        assert not y.any() and not dx.any()
        x = x.detach()
    f = R.drop_factor(64, 33, 65535 / 65536, 1)
    R.assert_close(ops.dropout(x, 65535 / 65536, 1), *_drop_bound(x, f, 1.0))


def test_dropped_values_are_zero_whatever_they_hold(cuda):
    f = R.drop_factor(200, 40, 0.5, 9)
    for bad in (float("inf"), float("-inf"), float("nan")):
        x = torch.ones(200, 40)
        x[f == 0] = bad
        x = x.cuda().requires_grad_()
        y = ops.dropout(x, 0.5, 9, negative_slope=0.1)
        g = torch.where(f == 0, bad, 1.0).float().cuda()
        dx, = torch.autograd.grad(y, x, g)
        assert torch.equal(y.detach().cpu(), (f / 1.0).float())
        assert torch.equal(dx.cpu(), f.float())
        # one that is kept stays what it is
        x = torch.where(f == 0, 1.0, bad).float().cuda()
        y = ops.dropout(x, 0.5, 9).cpu()
        assert not y[f == 0].any() and not torch.isfinite(y[f != 0]).any()


def test_dropout_views_and_ranks(cuda):
    wide = _randn(50, 200)
    f = R.drop_factor(50, 64, 0.3, 5)
    for x in (wide[:, 3:67], wide[:, 8:72], wide[:1, :64].expand(50, 64),
              wide[::2, :64].repeat(2, 1)[:50]):
        R.assert_close(ops.dropout(x, 0.3, 5), *_drop_bound(x, f, 1.0))
    x3 = _randn(5, 10, 64)
    assert torch.equal(ops.dropout(x3, 0.3, 5).view(50, 64), ops.dropout(x3.view(50, 64), 0.3, 5))
    x1 = _randn(64)
    assert torch.equal(ops.dropout(x1, 0.3, 5), ops.dropout(x1[None], 0.3, 5)[0])
    # an expanded gradient (a sum's)
    x = wide[:, 3:67].detach().requires_grad_()
    dx, = torch.autograd.grad(ops.dropout(x, 0.3, 5).sum(), x)
    assert torch.equal(dx.cpu(), f.float())
    # no rows
    e = torch.empty(0, 64, device="cuda", requires_grad=True)
    assert ops.dropout(e, 0.3, 5).shape == (0, 64)
    assert torch.autograd.grad(ops.dropout(e, 0.3, 5).sum(), e)[0].shape == (0, 64)
    # gradients of a broadcast input sum over its rows
    b = _randn(1, 64).requires_grad_()
    db, = torch.autograd.grad(ops.dropout(b.expand(50, 64), 0.3, 5).sum(), b)
    want = f.sum(0, keepdim=True)
    R.assert_close(db, want, 60 * R.U * want)


def test_dropout_places(cuda):
    """A value's fate is its place's: shards, far rows, sites and seeds."""
    x = _randn(100, 48)
    y = ops.dropout(x, 0.4, SEED)
    assert torch.equal(ops.dropout(x[37:], 0.4, SEED, row0=37), y[37:])
    far = 2 ** 33 + 5
    R.assert_close(ops.dropout(x, 0.4, SEED, row0=far),
                   *_drop_bound(x, R.drop_factor(100, 48, 0.4, SEED, row0=far), 1.0))
    seen = [y, ops.dropout(x, 0.4, SEED, site=1), ops.dropout(x, 0.4, SEED + 1),
            ops.dropout(x, 0.4, SEED + 2 ** 40)]
    for i, a in enumerate(seen):
        for b in seen[:i]:
            assert ((a == 0) != (b == 0)).float().mean() > 0.4
    neg = ops.dropout(x, 0.4, -7)                 # taken modulo 2^64
    assert torch.equal(neg, ops.dropout(x, 0.4, 2 ** 64 - 7))
    t = torch.tensor([-7], device="cuda")
    assert torch.equal(neg, ops.dropout(x, 0.4, t))
    assert torch.equal(neg, ops.dropout(x, 0.4, t[0]))


def test_dropout_past_32_bits(cuda):
    """A table of more than 2^31 elements: its last rows are those of a small call."""
    rows = 2 ** 31 // 64 + 1000
    x = torch.ones(rows, 64, dtype=BF16, device="cuda")
    y = ops.dropout(x, 0.5, 3)
    tail = ops.dropout(x[:300], 0.5, 3, row0=rows - 300)
    assert torch.equal(y[-300:], tail)
    x[-1, 0] = 1000.0
    z = ops.layer_norm(x)
    assert torch.equal(z[-300:], ops.layer_norm(x[-300:]))


# ---- layer norm and the block -------------------------------------------------------------
def _check_block(rows, d, dtype, wdtype, p, slope, with_res, with_w, shift=0.0, x=None):
    x = _randn(rows, d, dtype=dtype, shift=shift) if x is None else x
    res = _randn(rows, d, dtype=dtype, seed=1) if with_res else None
    w = _randn(d, dtype=wdtype, seed=2, shift=1.0) if with_w else None
    b = _randn(d, dtype=wdtype, seed=3) if with_w else None
    dy, dh = _randn(rows, d, dtype=dtype, seed=4), _randn(rows, d, dtype=dtype, seed=5)
    args = [t for t in (x, res, w, b) if t is not None]
    for t in args:
        t.requires_grad_()
    alone = p == 0 and slope == 1.0 and not with_res
    if alone:
        y = ops.layer_norm(x, w, b)
        got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, args, dy)))
    else:
        y, h = ops.dropout_add_layer_norm(x, res, w, b, p, SEED, site=2, negative_slope=slope)
        names = [n for n, t in (("dx", x), ("dres", res), ("dw", w), ("db", b)) if t is not None]
        got = dict(zip(names, torch.autograd.grad((y, h), args, (dy, dh))))
        got["h"] = h
    got["y"] = y
    cpu = [t.detach().cpu() if t is not None else None for t in (x, res, w, b)]
    f = (R.drop_factor(rows, d, p, SEED, site=2) if p
         else torch.ones(rows, d, dtype=torch.float64))
    want = R.block(*cpu, 1e-5, f, slope, dy.cpu(), None if alone else dh.cpu())
    for name, v in got.items():
        R.assert_close(v, *want[name], f"{name} {rows}x{d} {dtype}")


WIDTHS = [1, 2, 3, 7, 8, 9, 16, 17, 31, 32, 33, 64, 65, 100, 128, 129, 255, 256, 321, 512, 513, 1000, 1024, 1025,
          2048, 2049, 4096, 4097, 8192, 8193, 16384]


@pytest.mark.parametrize("d", WIDTHS)
def test_layer_norm_widths(cuda, d):
    _check_block(37, d, F32, F32, 0.0, 1.0, False, True)


@pytest.mark.parametrize("d", WIDTHS)
def test_block_widths(cuda, d):
    _check_block(11, d, F32, F32, 0.3, 0.2, True, True)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("half_weights", [True, False])
@pytest.mark.parametrize("rows,d", [(1, 64), (50, 201), (9, 1030), (5, 5000)])
def test_half_precision(cuda, dtype, half_weights, rows, d):
    wt = dtype if half_weights else F32
    _check_block(rows, d, dtype, wt, 0.0, 1.0, False, True)
    _check_block(rows, d, dtype, wt, 0.25, 0.01, True, True)


@pytest.mark.parametrize("with_res,with_w,p,slope", [
    (False, False, 0.0, 1.0), (False, False, 0.2, 0.2), (True, False, 0.0, 1.0),
    (True, True, 0.0, 0.2), (False, True, 0.5, 1.0), (True, True, 0.9, 1.0)])
def test_block_variants(cuda, with_res, with_w, p, slope):
    _check_block(70, 64, F32, F32, p, slope, with_res, with_w)


@pytest.mark.parametrize("rows", [1, 2, 31, 33, 1025, 5000, 40000])
def test_rows(cuda, rows):
    _check_block(rows, 40, F32, F32, 0.1, 0.2, True, True)


@pytest.mark.parametrize("d", [3, 8, 16, 30, 32])
@pytest.mark.parametrize("rows", [300, 5001, 70000])
def test_rows_of_few_values(cuda, rows, d):
    """Rows of one to four lanes: up to 256 of them in a workgroup's sums."""
    _check_block(rows, d, F32, F32, 0.1, 0.2, True, True)
    _check_block(rows, d, BF16, F32, 0.0, 1.0, False, True)


def test_far_mean_and_constant_rows(cuda):
    """A mean far above the deviation costs no more than the inputs' own resolution; a constant
    row is exactly the bias."""
    _check_block(20, 64, F32, F32, 0.0, 1.0, False, True, shift=3000.0)
    b = _randn(300)
    for c in (0.0, 1000.1, -3e4):
        x = torch.full((5, 300), c, device="cuda")
        y = ops.layer_norm(x, None, b)
        assert torch.equal(y, b.expand(5, 300))


@pytest.mark.parametrize("d", [48, 64, 201, 1500, 4096])
def test_non_finite_rows_stay_in_their_row(cuda, d):
    x = _randn(64, d)
    want = ops.layer_norm(x)
    for bad in (float("inf"), float("nan")):
        z = x.clone()
        z[10, 3] = bad
        y = ops.layer_norm(z)
        assert torch.isnan(y[10]).all()
        keep = torch.arange(64) != 10
        assert torch.equal(y[keep], want[keep])


def test_everything_dropped(cuda):
    """p = 1 leaves the residual alone; without one the row is empty: y is the bias."""
    x, res, b = _randn(9, 64).requires_grad_(), _randn(9, 64, seed=1), _randn(64, seed=2)
    y, h = ops.dropout_add_layer_norm(x, res, None, b, 1.0, 4)
    assert torch.equal(h, res) and torch.equal(y, ops.layer_norm(res, None, b))
    dx, = torch.autograd.grad(y.sum() + h.sum(), x)
    assert not dx.any()
    y, h = ops.dropout_add_layer_norm(x, None, None, b, 1.0, 4)
    assert not h.any() and torch.equal(y, b.expand(9, 64))


def test_block_mask_is_dropouts(cuda):
    """h - residual is ops.dropout's answer, at every way of sharing the rows out."""
    for d in (5, 64, 300, 3000):
        x = _randn(30, d)
        z = torch.zeros_like(x)
        _, h = ops.dropout_add_layer_norm(x, z, None, None, 0.4, SEED, site=9, row0=77,
                                          negative_slope=0.2)
        assert torch.equal(h, ops.dropout(x, 0.4, SEED, site=9, row0=77, negative_slope=0.2))


def test_partial_gradients(cuda):
    """Only y, only h, only some inputs: each as in the whole."""
    x, res = _randn(40, 64), _randn(40, 64, seed=1)
    w, b = _randn(64, seed=2), _randn(64, seed=3)
    dy, dh = _randn(40, 64, seed=4), _randn(40, 64, seed=5)

    def grads(need, outs):
        leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, res, w, b), need)]
        y, h = ops.dropout_add_layer_norm(*leaves, 0.2, 5, negative_slope=0.2)
        o = [(y, dy), (h, dh)]
        o = [o[i] for i in outs]
        return torch.autograd.grad([v for v, _ in o], [t for t, n in zip(leaves, need) if n],
                                   [g for _, g in o], allow_unused=True)

    whole = grads((1, 1, 1, 1), (0, 1))
    for i in range(4):
        need = [j == i for j in range(4)]
        assert torch.equal(grads(need, (0, 1))[0], whole[i])
    f = R.drop_factor(40, 64, 0.2, 5)
    only_h = grads((1, 1, 1, 1), (1,))
    assert torch.equal(only_h[1], dh)
    fx = f * torch.where(x.cpu() > 0, 1.0, 0.2)
    R.assert_close(only_h[0], dh.cpu().double() * fx, 5 * R.U * (dh.cpu().double() * fx).abs())
    assert not only_h[2].any() and not only_h[3].any()
    only_y = grads((1, 1, 1, 1), (0,))
    want = R.block(x.cpu(), res.cpu(), w.cpu(), b.cpu(), 1e-5, f, 0.2, dy.cpu())
    for name, v in zip(("dx", "dres", "dw", "db"), only_y):
        R.assert_close(v, *want[name], name)
    assert torch.equal(only_y[2], whole[2]) and torch.equal(only_y[3], whole[3])


def test_views_and_ranks(cuda):
    wide = _randn(60, 500)
    for x in (wide[:, 1:65], wide[:, 100:164], wide[:1, :64].expand(60, 64)):
        _check_block(60, 64, F32, F32, 0.0, 1.0, False, True, x=x.detach())
        _check_block(60, 64, F32, F32, 0.1, 0.2, True, True, x=x.detach())
    x = _randn(3, 4, 5, 64)
    assert torch.equal(ops.layer_norm(x), ops.layer_norm(x.view(60, 64)).view_as(x))
    for shape in ((64,), (3, 4, 5, 64)):          # gradients of other ranks
        x, dy = _randn(*shape).requires_grad_(), _randn(*shape, seed=1)
        y, h = ops.dropout_add_layer_norm(x, x.detach(), None, None, 0.2, 3, negative_slope=0.2)
        got = torch.autograd.grad((y, h, ops.dropout(x, 0.2, 3)), x, (dy, dy, dy))[0]
        x2 = x.detach().view(-1, 64).requires_grad_()
        y, h = ops.dropout_add_layer_norm(x2, x2.detach(), None, None, 0.2, 3,
                                          negative_slope=0.2)
        d2 = dy.view(-1, 64)
        want = torch.autograd.grad((y, h, ops.dropout(x2, 0.2, 3)), x2, (d2, d2, d2))[0]
        assert got.shape == shape and torch.equal(got.view(-1, 64), want)
    res = _randn(1, 64).requires_grad_()          # one residual row for all
    x = _randn(60, 64, seed=8)
    y, h = ops.dropout_add_layer_norm(x, res.expand(60, 64), None, None, 0.0, 0)
    dr, = torch.autograd.grad((y, h), res, (torch.zeros_like(y), torch.ones_like(h)))
    assert torch.equal(dr, torch.full_like(dr, 60.0))


def test_saved_tensor_hooks(cuda):
    """A hook may give a saved view back with another layout (as one kept on the host is)."""
    wide, wide2 = _randn(40, 200), _randn(40, 200, seed=1)
    dy = _randn(40, 64, seed=2)

    def grads():
        x, r = (t[:, 3:67].detach().requires_grad_() for t in (wide, wide2))
        y, h = ops.dropout_add_layer_norm(x, r, None, None, 0.2, 5, negative_slope=0.2)
        z = ops.dropout(x, 0.2, 5, negative_slope=0.2)
        return torch.autograd.grad((y, h, z), (x, r), (dy, dy, dy))

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        got = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone().t().contiguous().t()
                                                  if t.dim() == 2 else t, lambda t: t):
        other = grads()
    for a, b, c in zip(want, got, other):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_no_rows(cuda):
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    b = torch.ones(64, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()


@pytest.mark.parametrize("scale,eps", [(1e-12, 1e-5), (1e-12, 0.0), (1e-18, 0.0), (1e8, 1e-5),
                                       (3e15, 1e-5), (1e18, 0.0)])
def test_variances_over_the_range(cuda, scale, eps):
    """1 / sqrt at both ends of what fp32 holds, within the estimate's range and outside it (the
    exact root there). Products below 2^-126 keep 2^-149, which at 1e-18 (variance 1e-36) is
    1e-9 of them."""
    x = _randn(20, 128) * scale
    y = ops.layer_norm(x, eps=eps)
    f = torch.ones(20, 128, dtype=torch.float64)
    want, bound = R.block(x.cpu(), None, None, None, eps, f, 1.0)["y"]
    R.assert_close(y, want, bound, f"{scale} {eps}")
    # beyond it: a variance of zero without eps has no norm; an overflowing one gives 0
    z = ops.layer_norm(torch.full((1, 8), 3.0, device="cuda"), eps=0.0)
    assert z.isnan().all()
    big = torch.tensor([[3e38, -3e38] * 32], device="cuda")
    assert not ops.layer_norm(big).any()


def test_equal_inputs_give_equal_bits(cuda):
    x, w = _randn(20000, 72).requires_grad_(), _randn(72, seed=1).requires_grad_()
    dy = _randn(20000, 72, seed=2)
    first = torch.autograd.grad(ops.layer_norm(x, w), (x, w), dy)
    for _ in range(3):
        again = torch.autograd.grad(ops.layer_norm(x, w), (x, w), dy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_refusals(cuda):
    x = _randn(4, 64)
    bad = [
        (TypeError, lambda: ops.dropout(x.double(), 0.1, 0)),
        (TypeError, lambda: ops.layer_norm(x.int())),
        (ValueError, lambda: ops.dropout(x, -0.1, 0)),
        (ValueError, lambda: ops.dropout(x, float("nan"), 0)),
        (ValueError, lambda: ops.dropout(x, 0.1, 0, site=2 ** 32)),
        (ValueError, lambda: ops.dropout(x, 0.1, 0, row0=-1)),
        (ValueError, lambda: ops.dropout(x.t(), 0.1, 0)),
        (ValueError, lambda: ops.dropout(x[:, :0], 0.1, 0)),
        (ValueError, lambda: ops.dropout(x[0, 0], 0.1, 0)),
        (TypeError, lambda: ops.dropout(x, 0.1, torch.zeros(1, device="cuda"))),
        (TypeError, lambda: ops.dropout(x, 0.1, torch.zeros(2, device="cuda").long())),
        (ValueError, lambda: ops.dropout(x, 0.1, torch.tensor(3))),
        (ValueError, lambda: ops.layer_norm(x, torch.ones(63, device="cuda"))),
        (ValueError, lambda: ops.layer_norm(x, torch.ones(64))),
        (ValueError, lambda: ops.layer_norm(x, torch.ones(128, device="cuda")[::2])),
        (ValueError, lambda: ops.layer_norm(x, eps=-1e-5)),
        (TypeError, lambda: ops.layer_norm(x, torch.ones(64, device="cuda").half())),
        (TypeError, lambda: ops.layer_norm(x.half(), torch.ones(64, device="cuda").half(),
                                           torch.ones(64, device="cuda"))),
        (NotImplementedError, lambda: ops.layer_norm(_randn(1, 16385))),
        (ValueError, lambda: ops.dropout_add_layer_norm(x, x[:3], None, None, 0.1, 0)),
        (TypeError, lambda: ops.dropout_add_layer_norm(x, x.half(), None, None, 0.1, 0)),
        (ValueError, lambda: ops.dropout_add_layer_norm(x, x.cpu(), None, None, 0.1, 0)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    # a seed tensor that moved on between the passes would draw another mask: refused
    t = torch.tensor([5], device="cuda")
    y = ops.dropout(x.requires_grad_(), 0.1, t)
    t.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_c_entries_leave_what_is_not_theirs(cuda):
    """Columns behind d and rows behind `rows` of wider outputs stay as they were."""
    x = _randn(20, 64)
    for dtype, code in ((F32, 0), (BF16, 1)):
        xt = x.to(dtype)
        for d in (61, 64):
            out = torch.full((30, 80), 7.0, dtype=dtype, device="cuda")
            launch("gnnrec_dropout_forward", x.device, code, 20, d, xt.data_ptr(), 64,
                   out.data_ptr(), 80, 0.5, 3, None, 0, 0, 1.0)
            assert (out[20:] == 7).all() and (out[:, d:] == 7).all()
            assert torch.equal(out[:20, :d], ops.dropout(xt[:, :d], 0.5, 3))
            out.fill_(7.0)
            launch("gnnrec_layer_norm_forward", x.device, code, code, 20, d, xt.data_ptr(), 64,
                   None, 0, None, None, 1e-5, 0.0, 0, None, 0, 0, 1.0, out.data_ptr(), 80, None,
                   0)
            assert (out[20:] == 7).all() and (out[:, d:] == 7).all()
            assert torch.equal(out[:20, :d], ops.layer_norm(xt[:, :d]))


def test_other_streams(cuda):
    x, w = _randn(3000, 64).requires_grad_(), _randn(64, seed=1).requires_grad_()
    dy = _randn(3000, 64, seed=2)

    def both():
        y, h = ops.dropout_add_layer_norm(x, x.detach(), w, None, 0.2, 3, negative_slope=0.2)
        return (y.detach(), h.detach()) + torch.autograd.grad((y, h), (x, w), (dy, dy))

    want = both()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:                      # three calls at once
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_captured_training_step_draws_new_masks(cuda):
    """A captured forward and backward with the seed in device memory: each replay equals the
    eager step for its seed, with eager work between the replays; two graphs at a time."""
    x, res = _randn(500, 64), _randn(500, 64, seed=1)
    w, b = _randn(64, seed=2), _randn(64, seed=3)
    dy, dh = _randn(500, 64, seed=4), _randn(500, 64, seed=5)

    def step(seed):
        leaves = [t.detach().requires_grad_() for t in (x, res, w, b)]
        y, h = ops.dropout_add_layer_norm(*leaves, 0.3, seed, negative_slope=0.2)
        z = ops.dropout(y, 0.1, seed, site=1)
        return (z.detach(), h.detach()) + torch.autograd.grad((z, h), leaves, (dy, dh))

    seeds = [torch.tensor([100 * i], device="cuda") for i in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in seeds:
            step(s)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in seeds:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.add_(1)
            outs.append(step(s))
        graphs.append(g)
    for i in range(1, 5):
        for k in range(2):
            graphs[k].replay()
            torch.cuda.synchronize()
            want = step(100 * k + i)
            assert all(torch.equal(a, c) for a, c in zip(outs[k], want)), (i, k)


def test_second_derivatives_are_refused(cuda):
    x = _randn(4, 64).requires_grad_()
    dx, = torch.autograd.grad(ops.layer_norm(x).pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_library_is_native(cuda):
    assert "gfx950" in _lib.version()
