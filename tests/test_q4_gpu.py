"""4-bit item tables on the GPU: the quantiser exactly, the products within a derived bound."""
import pytest
import torch

import rowwise_ref as R
from src import ops
from src.ops.rowwise import launch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _table(n, k, seed=0):
    """Random codes (in the padding too) and scales over several powers of two."""
    g = torch.Generator().manual_seed(seed)
    G = -(-k // 32)
    codes = torch.randint(0, 256, (n, G * 16), dtype=torch.uint8, generator=g)
    scale = torch.exp2(torch.rand(n, G, generator=g) * 6 - 3).bfloat16()
    return ops.Q4Table(codes.cuda(), scale.cuda(), k)


def _check(x, table, out=None, what=""):
    """Every product of a code and x is exact in the sum's first step or split into exact parts;
    a group's sum has at most 32 products in up to three parts (96 additions), the groups add
    one product with the scale and one sum each, joined in any order: (100 + 2 G) U of the sum
    of magnitudes."""
    got = ops.q4_matmul(x, table) if out is None else out
    v = R.q4_values(table.codes, table.scale, table.k)
    xd = x.detach().cpu().double()
    bound = (100 + 2 * table.scale.shape[1]) * R.U * (xd.abs() @ v.abs().t())
    R.assert_close(got, xd @ v.t(), bound, what)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k", [(1, 1), (5, 31), (17, 32), (16, 33), (64, 64), (63, 96), (65, 100),
                                 (130, 128), (200, 160), (100, 200), (333, 256), (70, 288),
                                 (48, 513), (33, 1000), (20, 2048), (3, 5000), (257, 4096)])
@pytest.mark.parametrize("m", [1, 3, 16])
def test_products(cuda, dtype, n, k, m):
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype).cuda()
    _check(x, _table(n, k), what=f"{m}x{n}x{k}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m", [2, 4, 5, 8, 12, 17, 32, 33, 64, 100])
def test_users(cuda, dtype, m):
    for n, k in ((3706, 64), (500, 256), (40, 600)):
        x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype).cuda()
        _check(x, _table(n, k, seed=1), what=f"{m}x{n}x{k}")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m", [1, 4, 5, 20])
@pytest.mark.parametrize("n,k", [(16383, 257), (16384, 257), (65535, 64), (65536, 64),
                                 (65537, 33), (65600, 96), (65537, 150), (65600, 192),
                                 (65601, 224), (17000, 2048), (16400, 2080), (70000, 300),
                                 (4100, 4096), (200, 8192), (50, 16000)])
def test_ways_of_sharing_out(cuda, dtype, m, n, k):
    """Both sides of every border between the kernels, and every number of trailing groups with
    one tile and with four; the table's rows repeat, so the oracle stays small."""
    t = _table(256, k, seed=2)
    rep = -(-n // 256)
    big = ops.Q4Table(t.codes.repeat(rep, 1)[:n], t.scale.repeat(rep, 1)[:n], k)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype).cuda()
    got = ops.q4_matmul(x, big)
    _check(x, t, out=got[:, :256].contiguous() if n >= 256 else ops.q4_matmul(x, t))
    first = got[:, :256] if n >= 256 else got
    for r in range(0, n, 256):
        part = got[:, r:r + 256]
        assert torch.equal(part, first[:, :part.shape[1]]), r


def test_users_beyond_a_grid_row(cuda):
    x = torch.randn(3000, 64, generator=torch.Generator().manual_seed(0)).cuda()
    _check(x, _table(90, 64))


def test_range_of_x(cuda):
    """fp32 users over the type's range: all 24 bits of x count, and the result keeps the bound
    relative to its own magnitudes; zeros give exact zeros."""
    g = torch.Generator().manual_seed(5)
    t = _table(100, 96)
    for e in (-100, -60, -20, 0, 40, 90, 107):
        x = torch.randn(4, 96, generator=g) * 2.0 ** e
        _check(x.cuda(), t, what=f"2^{e}")
    x = (1 + torch.arange(96.0)[None] * 2 ** -20).repeat(2, 1)     # only the low bits differ
    _check(x.cuda(), t)
    assert not ops.q4_matmul(torch.zeros(3, 96, device="cuda"), t).any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k", [64, 300, 2080])
def test_non_finite_values(cuda, dtype, k):
    """An infinity or a NaN of one user reaches that user's scores as in the full product, in
    each of the kernels (by the width and the number of users)."""
    t = _table(80, k, seed=3)
    v = R.q4_values(t.codes, t.scale, k)
    for m in (1, 2, 7, 20):
        for bad in (float("inf"), float("-inf"), float("nan")):
            x = torch.randn(m, k, generator=torch.Generator().manual_seed(1)).to(dtype)
            clean = ops.q4_matmul(x.cuda(), t)
            x[m // 2, 40] = bad
            got = ops.q4_matmul(x.cuda(), t).cpu()
            want = (x[m // 2].double() @ v.t())
            assert torch.equal(got[m // 2].isnan(), want.isnan())
            inf = want.isinf()
            assert torch.equal(got[m // 2][inf].double(), want[inf])
            rest = torch.arange(m) != m // 2
            assert torch.equal(got[rest], clean.cpu()[rest])


def test_nan_payloads_and_scales(cuda):
    t = _table(80, 64, seed=3)
    # a NaN with only low payload bits, which half of a word would take for an infinity
    x = torch.zeros(1, 64)
    x.view(torch.int32)[0, 3] = 0x7F800001
    assert ops.q4_matmul(x.cuda(), t).isnan().all()
    # a NaN scale is its row's
    s = t.scale.clone()
    s[7, 1] = float("nan")
    got = ops.q4_matmul(torch.randn(5, 64, device="cuda"), ops.Q4Table(t.codes, s, 64))
    assert got[:, 7].isnan().all() and not got[:, torch.arange(80) != 7].isnan().any()


def test_views_and_output_types(cuda):
    t = _table(150, 100)
    wide = torch.randn(9, 333, generator=torch.Generator().manual_seed(2)).cuda()
    for x in (wide[:, 1:101], wide[::2, 7:107], wide[:1, :100].expand(6, 100)):
        _check(x, t)
    for dtype in (F32, BF16, F16):
        x = wide[:, :100].to(dtype)
        for out in (F32, BF16, F16):
            _check(x, t, out=ops.q4_matmul(x, t, out_dtype=out))
    one = ops.q4_matmul(wide[0, 3:103], t)
    assert one.shape == (150,)
    assert torch.equal(one, ops.q4_matmul(wide[:1, 3:103], t)[0])
    assert ops.q4_matmul(wide[:0, :100], t).shape == (0, 150)
    empty = ops.Q4Table(t.codes[:0], t.scale[:0], 100)
    assert ops.q4_matmul(wide[:, :100], empty).shape == (9, 0)
    off = torch.zeros(150 * 64 + 8, dtype=torch.uint8, device="cuda")[8:].view(150, 64)
    off.copy_(t.codes)                      # codes that are not 16-B aligned are copied once
    assert torch.equal(ops.q4_matmul(wide[:, :100], ops.Q4Table(off, t.scale, 100)),
                       ops.q4_matmul(wide[:, :100], t))


def test_output_rows_keep_their_neighbours(cuda):
    t = _table(75, 64)
    x = torch.randn(5, 64, device="cuda")
    out = torch.full((7, 90), 3.0, device="cuda")
    launch("gnnrec_q4_matmul", x.device, 0, 0, 5, x.data_ptr(), 64, 75, 64, t.codes.data_ptr(),
           t.scale.data_ptr(), out.data_ptr(), 90, None)
    assert (out[5:] == 3).all() and (out[:, 75:] == 3).all()
    assert torch.equal(out[:5, :75], ops.q4_matmul(x, t))


def test_many_items(cuda):
    """A catalogue of many thousand workgroups, and items past 2^31 bytes of codes."""
    n = 3_000_001
    t = _table(1 << 12, 64)
    rep = -(-n // (1 << 12))
    big = ops.Q4Table(t.codes.repeat(rep, 1)[:n], t.scale.repeat(rep, 1)[:n], 64)
    x = torch.randn(2, 64, device="cuda")
    got, want = ops.q4_matmul(x, big), ops.q4_matmul(x, t)
    assert torch.equal(got, want.repeat(1, rep)[:, :n])
    n, k = 1_100_000, 4096                  # 2.25e9 bytes
    t = _table(1 << 10, k)
    rep = -(-n // (1 << 10))
    big = ops.Q4Table(t.codes.repeat(rep, 1)[:n], t.scale.repeat(rep, 1)[:n], k)
    x = torch.randn(1, k, device="cuda").bfloat16()
    got = ops.q4_matmul(x, big, out_dtype=F32)
    v = R.q4_values(t.codes, t.scale, k)
    xd = x.cpu().double()
    bound = (100 + 2 * 128) * R.U * (xd.abs() @ v.abs().t())
    R.assert_close(got[:, -1024:].roll(n % 1024, 1), xd @ v.t(), bound)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (100, 32), (77, 33), (500, 64), (9, 1000)])
def test_quantize(cuda, dtype, n, k):
    w = (torch.randn(n, k, generator=torch.Generator().manual_seed(0)) * 0.1).to(dtype)
    t = ops.quantize_q4(w.cuda())
    codes, scale = R.q4_quantize(w)
    assert torch.equal(t.scale.cpu(), scale)
    assert torch.equal(t.codes.cpu(), codes)
    assert torch.equal(t.dequantize().cpu().double(), R.q4_values(codes, scale, k))


def test_quantize_borders(cuda):
    """Every border between two codes, a step below and above it, and special groups."""
    s = torch.tensor(0.37).bfloat16().float()          # the scale: the group's largest is 6 s
    vals = []
    for b in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
        t = b * s
        vals += [t, torch.nextafter(t, t * 0), torch.nextafter(t, t * 2)]
    row = torch.stack(vals + [6 * s] + [torch.tensor(0.0)] * 10)
    w = torch.stack([row, -row, row.flip(0)])
    t = ops.quantize_q4(w.cuda())
    codes, scale = R.q4_quantize(w)
    assert (scale.float() == s).all()
    assert torch.equal(t.codes.cpu(), codes) and torch.equal(t.scale.cpu(), scale)
    w = torch.zeros(6, 64)
    w[1, 3], w[2, 5], w[3, 40] = float("inf"), float("nan"), float("-inf")
    w[4, :32] = 1e-42                                  # scales below the normal range
    w[5, :] = 3e38
    t = ops.quantize_q4(w.cuda())
    codes, scale = R.q4_quantize(w)
    nan = scale.isnan()
    assert torch.equal(t.scale.cpu().isnan(), nan)
    assert torch.equal(t.scale.cpu()[~nan], scale[~nan]) and torch.equal(t.codes.cpu(), codes)
    assert nan.sum() == 3


def test_quantize_views(cuda):
    w = torch.randn(50, 300, device="cuda")
    for v in (w[:, 3:103], w[::3], w[:1].expand(20, 300)):
        t, u = ops.quantize_q4(v), ops.quantize_q4(v.clone())
        assert torch.equal(t.codes, u.codes) and torch.equal(t.scale, u.scale)
    t = ops.quantize_q4(w[:0])
    assert t.shape == (0, 300) and t.dequantize().shape == (0, 300)


def test_coarse_groups(cuda):
    """Scales of 64 and 128 columns stand for every 32 of them."""
    t = _table(40, 200)
    for group in (64, 128):
        s = t.scale[:, :-(-200 // group)].contiguous()
        wide = ops.Q4Table(t.codes, s, 200, group=group)
        x = torch.randn(2, 200, device="cuda")
        _check(x, wide)


def test_refusals(cuda):
    t = _table(10, 64)
    x = torch.randn(2, 64, device="cuda")
    for kind, call in ((ValueError, lambda: ops.q4_matmul(x.cpu(), t)),
                       (TypeError, lambda: ops.q4_matmul(x.double(), t)),
                       (ValueError, lambda: ops.q4_matmul(x[:, :63], t)),
                       (ValueError, lambda: ops.q4_matmul(x[None], t)),
                       (ValueError, lambda: ops.q4_matmul(torch.randn(64, 2).cuda().t(), t)),
                       (NotImplementedError,
                        lambda: ops.q4_matmul(x[:1].expand(65536, 64), t)),
                       (ValueError, lambda: ops.quantize_q4(x[0])),
                       (TypeError, lambda: ops.quantize_q4(x.long())),
                       (ValueError, lambda: ops.quantize_q4(x[:, :0]))):
        with pytest.raises(kind):
            call()


def test_streams_and_graphs(cuda):
    t = _table(5000, 160)
    x = torch.randn(4, 160, device="cuda")
    want = ops.q4_matmul(x, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.q4_matmul(x, t)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    w = torch.randn(5000, 160, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.q4_matmul(x, ops.quantize_q4(w))
    for i in range(4):
        w.normal_()
        x.normal_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.q4_matmul(x, ops.quantize_q4(w))), i
