"""The row-wise operators (dropout, layer norm, the block between two hops, 4-bit items) alone:
the calls of every case of perf/operators.py, and of those named in EXTRA, captured into a graph
with three rotating sets of inputs and replayed ("us", microseconds a pass), and as eager calls
on the same sets, waited for at the end ("call_us"). First the rates that their floors are stated
at: a copy of 2 GiB and a bfloat16 product of 8192^3.

    python tools/exp_row_operators.py                  # one JSON line each
    python tools/exp_row_operators.py --run "<case>"   # 12 eager passes of one case, for a profiler
"""
import importlib.util
import json
import os
import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
os.chdir(ROOT)
sys.path[:0] = [str(ROOT / "gnn-recommendations_amd"), str(ROOT)]
spec = importlib.util.spec_from_file_location("operator_cases", ROOT / "perf" / "operators.py")
cases = importlib.util.module_from_spec(spec)
spec.loader.exec_module(cases)
cases.own = True
from src import ops  # noqa: E402

cases._ops = lambda: ops     # (the cases look the package up in every pass)


def scores(m, n, k, kind):
    return {"name": f"scores {m} x {n} x {k} {kind}", "op": "scores", "m": m, "n": n, "k": k,
            "type": kind}


def norm(rows, d, kind):
    return {"name": f"norm {rows} x {d} {kind}", "op": "norm", "rows": rows, "d": d, "type": kind,
            "train": True}


# the products that no listed case reaches (more than four users, long rows), widths on both sides
# of a step in the lanes a row takes, and half-precision tables quantised
EXTRA = ([scores(*c) for c in ((16, 8192, 8192, "f32"), (16, 8192, 8192, "bf16"),
                               (64, 7812, 8192, "f32"), (64, 7812, 8192, "bf16"),
                               (1, 14336, 4096, "bf16"), (64, 1_000_000, 64, "f32"))]
         + [norm(r, d, k) for k in ("f32", "f16")
            for r, d in ((131072, 256), (131072, 257), (32768, 1024), (32768, 1025), (8192, 4096),
                         (8192, 4097))]
         + [{"name": f"quantize 1M items {k}", "op": "quantize", "n": 1_000_000, "k": 64,
             "type": k} for k in ("bf16", "f16")])
every = cases.listed() + EXTRA

if sys.argv[1:2] == ["--run"]:
    case = next(c for c in every if c["name"] == sys.argv[2])
    sets = [cases.prepare(case, i) for i in range(3)]
    for i in range(12):
        cases.run(sets[i % 3])
    torch.cuda.synchronize()
    print("done")
    sys.exit(0)


def host_time(f, n=20):
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) / n


x = torch.zeros(1 << 29, device="cuda")
y = torch.empty_like(x)
copy = 2 * x.numel() * 4 / host_time(lambda: y.copy_(x))
del x, y
a, b = (torch.randn(8192, 8192, device="cuda").bfloat16() for _ in range(2))
print(json.dumps({"copy_tb_s": round(copy / 1e12, 2), "bf16_product_tflops":
                  round(2 * 8192 ** 3 / host_time(lambda: a @ b) / 1e12)}), flush=True)
del a, b
for case in every:
    work = cases.work(case)
    sets = [cases.prepare(case, i) for i in range(3)]
    reps = max(1, min(20, int(2e9 / work["bytes"])))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            cases.run(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(reps):
            for s in sets:
                out = cases.run(s)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    times = []
    for _ in range(7):
        t0, t1 = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        t0.record()
        graph.replay()
        t1.record()
        torch.cuda.synchronize()
        times.append(t0.elapsed_time(t1) * 1e3 / (reps * 3))
    us = sorted(times)[3]
    turn = iter(range(10 ** 9))
    call = sorted(host_time(lambda: cases.run(sets[next(turn) % 3]), 60) for _ in range(7))[3]
    print(json.dumps({"case": case["name"], "us": round(us, 2), "call_us": round(call * 1e6, 1),
                      "case_tb_s": round(work["bytes"] / us / 1e6, 3),
                      "tflops": round(work["flops"] / us / 1e6, 1)}), flush=True)
    del sets, graph, out
    torch.cuda.empty_cache()
