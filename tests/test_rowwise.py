"""The row-wise operators where no GPU is needed: the generator's published answers, the plain
forms' gradients against differences, and everything that the entries refuse."""
import ctypes as C

import numpy as np
import pytest
import torch

import rowwise_ref as R
from src import ops
from src.ops import _lib


def test_philox_known_answers():
    """Philox4x32-10's known answers: all-zero and all-one counter and key, and digits of pi."""
    f = 0xFFFFFFFF
    for ctr, key, want in (
            ([0] * 4, [0] * 2, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
            ([f] * 4, [f] * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
            ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0],
             "d16cfe09 94fdcceb 5001e420 24126ea1")):
        got = R.philox4x32(np.array([ctr], np.uint64), key)[0]
        assert " ".join(f"{int(v):08x}" for v in got) == want


def test_drop_share():
    """The kept share is 1 - border / 65536 within five standard deviations."""
    for p in (0.1, 0.5, 0.9):
        kept = (R.drop_factor(500, 200, p, 7) != 0).double().mean()
        q = 1 - R.border_of(p) / 65536
        assert abs(float(kept) - q) < 5 * (q * (1 - q) / 1e5) ** 0.5


@pytest.mark.parametrize("slope,p", [(0.2, 0.3), (1.0, 0.0)])
def test_plain_gradients_against_differences(slope, p):
    """The oracle's gradients are those of the oracle's forward: central differences of step e
    along a random direction are off by e^2 / 6 times the third derivative (of order 1 / var,
    at most about 1e2 here), and by the rounding 2^-53 / e of a sum of about 1e3."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(6, 13, generator=g, dtype=torch.float64)
    x = torch.where(x.abs() < 1e-2, 0.1, x)     # away from the LeakyReLU's corner
    res, dy, dh = (torch.randn(6, 13, generator=g, dtype=torch.float64) for _ in range(3))
    w, b = (torch.randn(13, generator=g, dtype=torch.float64) for _ in range(2))
    f = R.drop_factor(6, 13, p, 11)
    out = R.block(x, res, w, b, 1e-5, f, slope, dy, dh)

    def loss(x, res, w, b):
        o = R.block(x, res, w, b, 1e-5, f, slope)
        return float((o["y"][0] * dy).sum() + (o["h"][0] * dh).sum())

    e = 1e-4
    args = [x, res, w, b]
    for i, name in enumerate(("dx", "dres", "dw", "db")):
        v = torch.randn(args[i].shape, generator=g, dtype=torch.float64)
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + e * v, args[i] - e * v
        diff = (loss(*up) - loss(*dn)) / (2 * e)
        assert abs(diff - float((out[name][0] * v).sum())) < 1e-5


def test_cpu_tensors_are_refused():
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.dropout(x, 0.1, 1)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.layer_norm(x)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.dropout_add_layer_norm(x, x, None, None, 0.1, 1)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.quantize_q4(x)
    t = ops.Q4Table(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 1).bfloat16(), 8)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.q4_matmul(x, t)
    with pytest.raises(ValueError, match="ROCm device"):
        t.dequantize()


def test_q4_table_refusals():
    codes = torch.zeros(4, 32, dtype=torch.uint8)
    scale = torch.zeros(4, 2).bfloat16()
    assert ops.Q4Table(codes, scale, 40).shape == (4, 40)
    assert ops.Q4Table(codes, scale[:, :1], 40, group=64).scale.shape == (4, 2)
    assert ops.Q4Table(codes, scale, 64).nbytes == 4 * 36
    for bad in (lambda: ops.Q4Table(codes, scale, 65), lambda: ops.Q4Table(codes, scale, 32),
                lambda: ops.Q4Table(codes, scale, 0), lambda: ops.Q4Table(codes[:3], scale, 64),
                lambda: ops.Q4Table(codes, scale, 64, group=16),
                lambda: ops.Q4Table(codes, scale, 64, group=64),
                lambda: ops.Q4Table(codes[0], scale, 64)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.Q4Table(codes.int(), scale, 64),
                lambda: ops.Q4Table(codes, scale.float(), 64)):
        with pytest.raises(TypeError):
            bad()
    t = ops.Q4Table(codes, scale, 64)
    with pytest.raises(TypeError):
        ops.q4_matmul(torch.zeros(1, 64), codes)
    with pytest.raises(TypeError):
        ops.q4_matmul(torch.zeros(1, 64), t, out_dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.q4_matmul(torch.zeros(1, 63), t)


def _err(rc):
    return rc, _lib.lib().gnnrec_last_error().decode()


def test_c_entries_refuse_before_they_launch():
    """Every refusal is the host's: these calls run without a GPU. The pointers are never read."""
    L = _lib.lib()
    buf = (C.c_float * 64)()
    a = (C.addressof(buf) + 15) & ~15       # 16-B aligned

    def drop(dtype=0, rows=2, d=8, x=a, y=a, p=0.5, row0=0):
        return _err(L.gnnrec_dropout_forward(dtype, rows, d, x, d, y, d, p, 1, None, 0, row0, 0.2,
                                             None))

    for kw, word in ((dict(dtype=3), "dtype"), (dict(rows=-1), "size"), (dict(d=0), "size"),
                     (dict(x=None), "null"), (dict(y=None), "null"), (dict(p=1.5), "p must"),
                     (dict(p=float("nan")), "p must"), (dict(row0=-1), "row0"),
                     (dict(rows=2 ** 60), "large")):
        rc, msg = drop(**kw)
        assert rc == -1 and word in msg, (kw, msg)
    assert drop(rows=0, x=None, y=None)[0] == 0
    # x is needed where the activation's sign is
    rc = L.gnnrec_dropout_backward(0, 2, 8, None, 0, a, 8, a, 8, 0.5, 1, None, 0, 0, 0.2, None)
    assert rc == -1

    def norm(dtype=0, wdtype=0, rows=2, d=8, x=a, y=a, eps=1e-5, p=0.0):
        return _err(L.gnnrec_layer_norm_forward(dtype, wdtype, rows, d, x, d, None, 0, None, None,
                                                eps, p, 0, None, 0, 0, 1.0, y, d, None, d, None))

    for kw, want in ((dict(dtype=-1), -1), (dict(wdtype=1), -1), (dict(dtype=1, wdtype=2), -1),
                     (dict(rows=-1), -1), (dict(d=0), -1), (dict(d=16385), -3),
                     (dict(x=None), -1), (dict(y=None), -1), (dict(eps=-1.0), -1),
                     (dict(eps=float("nan")), -1), (dict(p=-0.1), -1), (dict(rows=2 ** 40), -1)):
        assert norm(**kw)[0] == want, kw
    assert norm(rows=0, x=None, y=None)[0] == 0
    # a weight gradient needs its workspace
    rc = L.gnnrec_layer_norm_backward(0, 0, 2, 8, a, 8, None, 0, None, 1e-5, 0.0, 0, None, 0, 0,
                                      1.0, a, 8, None, 0, None, 8, None, 8, a, None, None, None)
    assert rc == -1
    assert L.gnnrec_layer_norm_work_floats(5, 64) == 2 * 64
    assert L.gnnrec_layer_norm_work_floats(0, 64) == 0

    def q4(dtype=0, out=0, m=1, n=4, k=64, codes=a, x=a, o=a, work=None):
        return _err(L.gnnrec_q4_matmul(dtype, out, m, x, k, n, k, codes, a, o, n, work, None))

    for kw, word in ((dict(dtype=7), "dtype"), (dict(out=7), "dtype"), (dict(m=-1), "rows"),
                     (dict(m=65536), "65535"), (dict(n=-1), "size"), (dict(k=0), "size"),
                     (dict(k=2 ** 30), "size"), (dict(codes=None), "null"),
                     (dict(codes=a + 4), "aligned"), (dict(x=None), "null"),
                     (dict(o=None), "null"), (dict(n=2 ** 50), "large"),
                     (dict(m=5, k=257), "workspace"),
                     (dict(m=5, k=257, work=a + 4), "workspace")):
        rc, msg = q4(**kw)
        assert rc == -1 and word in msg, (kw, msg)
    assert q4(n=0)[0] == 0 and q4(m=0)[0] == 0
    work = L.gnnrec_q4_matmul_work_bytes
    assert [work(t, 5, 4, k) for t in (0, 1, 2) for k in (256, 257)] \
        == [0, 3 * 5 * 288 * 2, 0, 5 * 288 * 2, 0, 2 * 5 * 288 * 2]
    assert work(1, 5, 4, 512) == 0 and work(0, 4, 4, 257) == 0 and work(9, 5, 4, 257) == 0
    assert L.gnnrec_quantize_q4(0, 4, 64, None, 64, a, a, None) == -1
    assert L.gnnrec_quantize_q4(9, 4, 64, a, 64, a, a, None) == -1
    assert L.gnnrec_dequantize_q4(4, 64, a, a, None, 64, None) == -1
