"""4-bit products where one tile holds the whole table, and each kernel on several streams and in
captured graphs."""
import pytest
import torch

from src import ops
from test_q4_gpu import BF16, F16, F32, _check, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m", [1, 4, 5, 20])
@pytest.mark.parametrize("n,k", [(200, 8192), (50, 16000), (9, 8192), (1, 2080), (255, 300)])
def test_partial_last_tiles_of_long_rows(cuda, dtype, m, n, k):
    """Tables whose last (or only) tile is partial, against the oracle itself."""
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(dtype).cuda()
    _check(x, _table(n, k, seed=2), what=f"{m}x{n}x{k}")


# one case a kernel: rows walked alone, split rows, split rows with the users cut into a workspace
WAYS = [(4, 160), (20, 160), (4, 1000), (20, 2080), (5, 300)]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("m,k", WAYS)
def test_streams(cuda, dtype, m, k):
    """Calls of their own users on several streams at once, again and again: none takes what
    another has in its workspace."""
    t = _table(4000, k)
    xs = [torch.randn(m, k, generator=torch.Generator().manual_seed(i)).to(dtype).cuda()
          for i in range(4)]
    want = [ops.q4_matmul(x, t) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.q4_matmul(xs[i], t))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(v, w) for v in g)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("m,k", WAYS)
def test_graphs(cuda, dtype, m, k):
    """Two captured graphs replayed in turn, with eager calls between the replays."""
    xs = [torch.randn(m, k, device="cuda").to(dtype) for _ in range(2)]
    ws = [torch.randn(3000, k, device="cuda").to(dtype) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.q4_matmul(xs[0], ops.quantize_q4(ws[0]))
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x, w in zip(xs, ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.q4_matmul(x, ops.quantize_q4(w)))
        graphs.append(g)
    for i in range(4):
        for x, w in zip(xs, ws):
            x.normal_()
            w.normal_()
        for g in graphs:
            g.replay()
        for x, w, out in zip(xs, ws, outs):
            assert torch.equal(out, ops.q4_matmul(x, ops.quantize_q4(w))), i
        torch.cuda.synchronize()
