"""The row-wise operators inside the framework's own paths: NGCF's counter-based dropout and
layer norm, ranking against 4-bit items, and a run of them together."""
import os

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
import torch.nn.functional as F

import rowwise_ref as R
from test_distributed import _free_port, cpu_ngcf_layer
from test_models import torch_adj

from src import ops
from src.data.dataset import RecommendationDataset
from src.evaluation import Evaluator
from src.models import NGCF, NGCFGroupShuffle
from src.ops import CsrGraph


def _model(cls=NGCF, seed=5, sizes=(64, 64, 32), **kw):
    torch.manual_seed(seed)
    m = cls(300, 500, embedding_dim=64, layer_sizes=list(sizes), dropout=0.1, init_scale=0.3,
            **kw)
    with torch.no_grad():
        for layer in m.layers:
            for lin in (layer.W1, layer.W2):
                lin.bias.normal_(std=0.1)
            if layer.norm is not None:
                layer.norm.weight.normal_(1.0, 0.2)
                layer.norm.bias.normal_(std=0.2)
    return m


def _composed(m, adj, masks=None):
    """NGCF's forward from elementary torch operations in 64 bits; masks: [factors] a layer."""
    x = m._initial_table()
    outs = [x]
    for k, layer in enumerate(m.layers):
        n = adj @ x
        z = F.leaky_relu(layer.W1(n) + layer.W2(x * n), 0.2)
        if masks is not None:
            z = z * masks[k]
        if layer.norm is not None:
            h = x + z if x.shape == z.shape else z
            z = F.layer_norm(h, (h.shape[1],), layer.norm.weight, layer.norm.bias)
        x = z
        outs.append(x)
    return torch.cat(outs, dim=1)


def _double(m, **kw):
    d = _model(type(m), **kw).double()
    d.load_state_dict({k: v.detach().cpu().double() for k, v in m.state_dict().items()})
    return d


def test_options_are_off_and_add_nothing():
    plain, torch_default = _model(), NGCF(300, 500)
    assert all(layer.norm is None and not layer.counter_dropout for layer in torch_default.layers)
    with_norm = _model(layer_norm=True)
    extra = set(with_norm.state_dict()) - set(plain.state_dict())
    assert extra == {f"layers.{k}.norm.{n}" for k in range(3) for n in ("weight", "bias")}
    assert torch.equal(with_norm.user_embedding.weight, plain.user_embedding.weight)


@pytest.mark.parametrize("cls", [NGCF, NGCFGroupShuffle])
def test_cpu_forward_with_layer_norm(cls):
    m = _model(cls, layer_norm=True, counter_dropout=True).eval()
    adj, nu, _ = torch_adj()
    with torch.no_grad():
        u, i = m(adj)
        assert u.shape == (300, 64 * 3 + 32) and torch.isfinite(u).all()
        if cls is NGCF:
            want = _composed(_double(m, layer_norm=True), adj.to_dense().double())
            # fp32 through three layers against 64 bits
            torch.testing.assert_close(torch.cat([u, i]).double(), want, rtol=1e-4, atol=1e-4)
    m.train()
    u, _ = m(adj)
    u.sum().backward()
    assert all(p.grad is not None for p in m.layers.parameters())


def _shard_worker(rank, world, port, q):
    from src.ops.distributed import DistributedGraph, ngcf_forward_dist
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        g, adj = _graph()
        with torch.no_grad():
            got = []
            for cls in (NGCF, NGCFGroupShuffle):
                m = _model(cls, layer_norm=True).eval()
                dg = DistributedGraph(g, rank, world, "cpu")
                whole = ngcf_forward_dist(dg, m, dg.pad_table(m._initial_table()),
                                          layer_fn=cpu_ngcf_layer, gather_output=True)
                got.append((whole.numpy(), torch.cat(m(adj)).numpy()))
            if rank == 0:
                q.put(got)
    finally:
        dist.destroy_process_group()


def test_sharded_forward_with_layer_norm():
    """Two ranks: the norm is row-local, so the shards give the rows of one device."""
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_shard_worker, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = q.get(timeout=120)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for whole, single in got:     # the stand-in layer sums in another order: fp32, three layers
        np.testing.assert_allclose(whole, single, rtol=1e-4, atol=1e-4)


def test_evaluator_refuses():
    with pytest.raises(ValueError, match="ROCm device"):
        Evaluator(device=torch.device("cpu"), item_bits=4)
    with pytest.raises(ValueError, match="4 or 32"):
        Evaluator(device=torch.device("cpu"), item_bits=8)


# ---- on the GPU ---------------------------------------------------------------------------
def _graph():
    adj, nu, ni = torch_adj()
    g = CsrGraph.from_torch_sparse(adj.coalesce())
    return g, adj


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(counter_dropout=True), dict(layer_norm=True),
                                dict(counter_dropout=True, layer_norm=True)])
def test_ngcf_training_matches_its_masks(cuda, kw):
    """Forward and every gradient of a training step, against the composition in 64 bits with
    the masks that the seed stands for."""
    g, adj = _graph()
    m = _model(**kw).to(cuda).train()
    m.dropout_seed = torch.tensor([77], device=cuda)
    out = torch.cat(m(g.to(cuda)))
    wgt = torch.randn(out.shape, generator=torch.Generator().manual_seed(1))
    (out * wgt.to(cuda)).sum().backward()

    d = _double(m, **kw)
    masks = [R.drop_factor(800, w, 0.1, 77, site=k) for k, w in enumerate((64, 64, 32))]
    want = _composed(d, adj.to_dense().double(), masks)
    (want * wgt.double()).sum().backward()
    # fp32 through three layers (Linear sums of 64, a hop, a norm) against 64 bits: relative to
    # the tensor's scale
    def off(a, b):
        return float((a.detach().cpu().double() - b).norm() / b.norm())
    assert off(out, want.detach()) < 1e-5
    for (name, p), q in zip(m.named_parameters(), d.parameters()):
        assert off(p.grad, q.grad) < 1e-4, name


@pytest.mark.gpu
def test_ngcf_seed_comes_from_torch(cuda):
    g, _ = _graph()
    g = g.to(cuda)
    m = _model(counter_dropout=True).to(cuda).train()
    outs = []
    for seed in (1, 1, 2):
        torch.manual_seed(seed)
        outs.append(torch.cat(m(g)).detach())
    assert torch.equal(outs[0], outs[1]) and not torch.equal(outs[0], outs[2])
    with pytest.raises(ValueError, match="needs a seed"):
        m.layers[0](m._initial_table(), g)
    m.eval()
    with torch.no_grad():
        plain = _model().to(cuda).eval()
        assert torch.equal(torch.cat(m(g)), torch.cat(plain(g)))


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [NGCF, NGCFGroupShuffle])
def test_ngcf_layer_norm_inference(cuda, cls):
    """The inference path (fused layer kernel, then the norm) and the training path with the
    dropout off are the same model, and the CPU's."""
    g, adj = _graph()
    g = g.to(cuda)
    m = _model(cls, layer_norm=True).to(cuda).eval()
    with torch.no_grad():
        fast = torch.cat(m(g))
    slow = torch.cat(m(g)).detach()
    torch.testing.assert_close(fast, slow, rtol=1e-4, atol=1e-5)
    cpu = _model(cls, layer_norm=True)
    cpu.load_state_dict({k: v.cpu() for k, v in m.state_dict().items()})
    with torch.no_grad():
        torch.testing.assert_close(fast.cpu(), torch.cat(cpu.eval()(adj)), rtol=1e-3, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [NGCF, NGCFGroupShuffle])
def test_one_rank_shard_with_layer_norm(cuda, cls):
    """A one-rank shard's native forward gives the rows of the model's own."""
    from src.ops.distributed import DistributedGraph, ngcf_forward_dist
    g, _ = _graph()
    g = g.to(cuda)
    dg = DistributedGraph(g, 0, 1, cuda)
    with torch.no_grad():
        m = _model(cls, sizes=(64, 64), layer_norm=True).to(cuda).eval()
        local = ngcf_forward_dist(dg, m, dg.pad_table(m._initial_table()))
        assert torch.equal(local[:800], torch.cat(m(g)))
        m = _model(cls, layer_norm=True).to(cuda).eval()
        with pytest.raises(NotImplementedError):     # a shard's layers keep their width
            ngcf_forward_dist(dg, m, dg.pad_table(m._initial_table()))


@pytest.mark.gpu
def test_rank_against_4_bit_items(cuda):
    """The ranking of the values that the codes stand for: exact order away from ties."""
    torch.manual_seed(3)
    users, items = torch.randn(150, 64, device=cuda), torch.randn(900, 64, device=cuda)
    rng = np.random.default_rng(0)
    seen = [np.sort(rng.choice(900, rng.integers(0, 40), replace=False)) for _ in range(150)]
    ptr = np.concatenate([[0], np.cumsum([len(s) for s in seen])]).astype(np.int64)
    col = np.concatenate(seen).astype(np.int32)
    got = Evaluator(device=cuda, item_bits=4).topk(users, items, list(range(150)), 20, ptr, col)
    table = ops.quantize_q4(items)
    v = R.q4_values(table.codes, table.scale, 64)
    score = users.cpu().double() @ v.t()
    for u in range(150):
        score[u, seen[u]] = float("-inf")
    best = score.topk(20, dim=1).values
    took = score.gather(1, got.cpu())
    # a neighbour may change places with one that is as good within the products' rounding
    assert torch.isfinite(took).all() and (took - best).abs().max() < 1e-4
    full = Evaluator(device=cuda).topk(users, items, list(range(150)), 20, ptr, col)
    share = np.mean([len(set(a.tolist()) & set(b.tolist())) / 20 for a, b in zip(got, full)])
    assert share > 0.5          # random embeddings, a tenth of the values' size lost


@pytest.mark.gpu
def test_train_then_serve_in_4_bits(cuda):
    """All of them as they are used together: NGCF with both options trained for an epoch,
    evaluated with full and with 4-bit items, one user scored."""
    from src.training import Trainer
    ds = RecommendationDataset.synthetic_movielens(n_users=200, n_items=300, n_ratings=6000,
                                                   seed=4)
    torch.manual_seed(0)
    m = NGCF(ds.n_users, ds.n_items, 64, [64, 64], 0.1, 0.1, counter_dropout=True,
             layer_norm=True)
    t = Trainer(m, ds, dict(batch_size=512, epochs=1, learning_rate=5e-3, use_scheduler=False,
                            warmup_epochs=0), device=cuda)
    before = [p.detach().clone() for p in m.parameters()]
    assert np.isfinite(t.train_epoch())
    assert all(not torch.equal(a, p) for a, p in zip(before, m.parameters()))
    full = Evaluator(device=cuda).evaluate(m, ds, adj_matrix=t.adj)
    four = Evaluator(device=cuda, item_bits=4).evaluate(m, ds, adj_matrix=t.adj)
    assert set(full) == set(four) and all(np.isfinite(v) for v in four.values())
    with torch.no_grad():
        users, items = m.get_all_embeddings(t.adj)
        table = ops.quantize_q4(items)
        one = ops.q4_matmul(users[7], table)
        want = users[7].cpu().double() @ R.q4_values(table.codes, table.scale, 192).t()
    bound = 120 * R.U * (users[7].abs().cpu().double()
                         @ R.q4_values(table.codes, table.scale, 192).abs().t())
    R.assert_close(one, want, bound)


@pytest.mark.gpu
def test_captured_ngcf_forward_draws_new_masks(cuda):
    """A captured training forward with the model's seed in device memory."""
    g, _ = _graph()
    g = g.to(cuda)
    m = _model(counter_dropout=True, layer_norm=True).to(cuda).train()
    m.dropout_seed = torch.tensor([10], device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad():
        with torch.cuda.stream(side):
            torch.cat(m(g))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            m.dropout_seed.add_(1)
            out = torch.cat(m(g))
        eager = _model(counter_dropout=True, layer_norm=True).to(cuda).train()
        for i in range(1, 5):
            graph.replay()
            torch.cuda.synchronize()
            eager.dropout_seed = torch.tensor([10 + i], device=cuda)
            assert torch.equal(out, torch.cat(eager(g))), i
