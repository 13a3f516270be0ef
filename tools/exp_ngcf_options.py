"""NGCF's BPR training step (K = 3, d = 64, batch 2048) with its row-wise options: the plain form
(torch's dropout), counter_dropout and layer_norm, each twice in turn in one process. Median ms a
step and the peak of allocated memory over the steps.

    python tools/exp_ngcf_options.py          # G100M (1M x 1M, 100M edges)
    python tools/exp_ngcf_options.py --ml1m   # the ML-1M shape
"""
import json
import sys
import time
from pathlib import Path

import numpy as np
import torch

ROOT = Path(__file__).resolve().parents[1]
sys.path[:0] = [str(ROOT / "gnn-recommendations_amd"), str(ROOT)]
import bench  # noqa: E402
from src.data.dataset import RecommendationDataset  # noqa: E402
from src.models import NGCF  # noqa: E402
from src.training import BPRLoss, DeviceSampler, make_adam, train_step  # noqa: E402

dev = torch.device("cuda", 0)
if "--ml1m" in sys.argv:
    ds = RecommendationDataset.synthetic_movielens(6040, 3706, 1_000_209, seed=1, name="ml-1m")
    g, nu, ni, warm, steps = ds.get_graph(dev), ds.n_users, ds.n_items, 10, 100
else:
    nu = ni = 1_000_000
    g, warm, steps = bench.build_graph(nu, ni, 100_000_000, 0, 16).to(dev), 2, 7
rp = g.row_ptr.cpu().numpy()
users = np.repeat(np.arange(nu), np.diff(rp[:nu + 1]))
items = g.col.cpu().numpy()[:rp[nu]] - nu
forms = {"plain": {}, "counter_dropout": {"counter_dropout": True}, "layer_norm":
         {"layer_norm": True}}
for name in [*forms, *forms]:
    torch.manual_seed(0)
    m = NGCF(nu, ni, 64, [64, 64, 64], **forms[name]).to(dev).train()
    samp = DeviceSampler(users, items, ni, 2048, 1, dev, seed=0)
    opt = make_adam(m.parameters(), 1e-3, 1e-4, dev)
    loss_fn = BPRLoss()
    for _ in range(warm):
        train_step(m, g, *samp(), opt, loss_fn, 1.0)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    ts = []
    for _ in range(steps):
        t0 = time.perf_counter()
        train_step(m, g, *samp(), opt, loss_fn, 1.0)
        torch.cuda.synchronize()
        ts.append((time.perf_counter() - t0) * 1e3)
    ts.sort()
    print(json.dumps({"users": nu, "items": ni, "form": name, "ms_median": round(ts[steps // 2], 3),
                      "ms_min": round(ts[0], 3),
                      "peak_gb": round(torch.cuda.max_memory_allocated() / 1e9, 2)}), flush=True)
    del m, opt
    torch.cuda.empty_cache()
