"""Plain 64-bit forms of the row-wise operators (dropout, layer norm, the block between two
hops, 4-bit tables) and the error bounds their fp32 kernels are held to."""
import numpy as np
import torch

U = 2.0 ** -24                                   # half a step of fp32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half of the smallest subnormal step: what a rounding adds near zero
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
E2M1 = np.array([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6])


def philox4x32(counter, key, rounds=10):
    """Philox4x32 of an [n, 4] array of counters (uint64 holding 32-bit words)."""
    m = np.uint64(0xFFFFFFFF)
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & m,
             (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return np.stack(c, axis=1)


def border_of(p):
    return int(np.floor(p * 65536 + 0.5))


def drop_factor(rows, d, p, seed, site=0, row0=0):
    """[rows, d] float64: 65536 / (65536 - border) where a value is kept, 0 where dropped."""
    nb = -(-d // 8)
    r = np.repeat(np.arange(rows, dtype=np.uint64) + np.uint64(row0), nb)
    ctr = np.stack([np.tile(np.arange(nb, dtype=np.uint64), rows), r & np.uint64(0xFFFFFFFF),
                    r >> np.uint64(32), np.full(rows * nb, site, np.uint64)], axis=1)
    seed = int(seed) % 2 ** 64
    w = philox4x32(ctr, (seed % 2 ** 32, seed >> 32))
    bits = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], axis=2).reshape(rows, nb * 8)
    b = border_of(p)
    keep = bits[:, :d].astype(np.int64) >= b
    return torch.from_numpy(keep * (65536.0 / (65536 - b) if b < 65536 else 0.0))


def leaky(x, slope):
    return torch.where(x > 0, x, x * slope)


def block(x, res, w, b, eps, f, slope, dy=None, dh=None):
    """Everything of the block in 64 bits, with each value's error bound: {name: (value,
    bound)}. x, res, dy, dh [rows, d]; w, b [d] or None; f: drop_factor's array.

    The bounds, U = 2^-24. A sum of a row goes through at most 38 additions (16 in a lane, 6 or
    10 across lanes, 16 across waves), so its error is at most 39 U times the sum of magnitudes.
    * h: the activation, the mask's scale (itself rounded), their product and the sum: 5 U
      of |act| + |h|.
    * xhat = (c - off) r with c = h - mean rounded (U |c|), off 39 U of mean |c| (at most the
      deviation, 1 in units of xhat), r half of the variance's 43 U plus the root and the
      quotient: together at most 64 U (1 + |xhat|), and h's own error times r, its mean over
      the row, and xhat times the mean of its product with xhat (the derivative of the norm).
    * dh = r (g - mean g - xhat mean(g xhat)): 64 U of the terms' magnitudes, and xhat's error
      in the last.
    """
    d = x.shape[1]
    x = x.double()
    a = leaky(x, slope)
    h = torch.where(f != 0, a * f, torch.zeros_like(a))
    act = h.abs()
    if res is not None:
        h = h + res.double()
    plain = res is None and slope == 1.0 and bool((f == 1).all())
    eh = torch.zeros_like(h) if plain else 5 * U * (act + h.abs())
    c = h - h.mean(1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    xhat = c * r
    ex = (64 * U * (1 + xhat.abs()) + r * (eh + eh.mean(1, keepdim=True)
          + xhat.abs() * (eh * xhat.abs()).mean(1, keepdim=True)))
    w1 = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b1 = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = xhat * w1 + b1
    out = {"h": (h, eh), "y": (y, ex * w1.abs() + 2 * U * y.abs())}
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w1
    m1, m2 = g.mean(1, keepdim=True), (g * xhat).mean(1, keepdim=True)
    a1, a2 = g.abs().mean(1, keepdim=True), (g * xhat).abs().mean(1, keepdim=True)
    ln = r * (g - m1 - xhat * m2)
    e = r * (64 * U * (g.abs() + a1 + xhat.abs() * (a2 + m2.abs())) + ex * m2.abs()
             + xhat.abs() * (g.abs() * ex).mean(1, keepdim=True))
    # r's own relative error: 24 U, and h's through the variance
    e = e + ln.abs() * (24 * U + r * (eh * xhat.abs()).mean(1, keepdim=True))
    dht = ln if dh is None else ln + dh.double()
    e = e + U * dht.abs()
    fx = f * torch.where(x > 0, 1.0, slope)
    out["dres"] = (dht, e)
    out["dx"] = (dht * fx, e * fx.abs() + 5 * U * (dht * fx).abs())
    # a column's sum: the rows of one lane group, the groups, the partial rows
    chain = x.shape[0] // 1024 + 64
    out["dw"] = ((dy * xhat).sum(0), (dy.abs() * ex).sum(0) + chain * U * (dy * xhat).abs().sum(0))
    out["db"] = (dy.sum(0), chain * U * dy.abs().sum(0))
    return out


def assert_close(got, want, bound, what=""):
    """got within the bound of want, plus its type's own rounding."""
    t = got.dtype
    got, want, bound = got.detach().cpu().double(), want.cpu(), bound.cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    tol = bound * (1 + 2 * HALF_STEP[t]) + HALF_STEP[t] * want.abs() + TINY[t]
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        i = int(torch.where(bad, ((got - want).abs() / tol).nan_to_num(9e9), 0).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values; at {i}: "
                             f"{got.flatten()[i]} for {want.flatten()[i]}, tolerance "
                             f"{tol.flatten()[i]}")


# ---- 4-bit tables -------------------------------------------------------------------------
def q4_quantize(w):
    """(codes uint8 [n, 16 G], scale bfloat16 [n, G]) of a float table, decided in 64 bits."""
    w = w.detach().cpu().double()
    n, k = w.shape
    G = -(-k // 32)
    v = torch.zeros(n, G * 32, dtype=torch.float64)
    v[:, :k] = w
    v = v.view(n, G, 32)
    scale = (v.abs().amax(2) / 6).float().bfloat16()
    finite = torch.isfinite(v).all(2)
    scale = torch.where(finite, scale, torch.full_like(scale, float("nan")))
    s = scale.double()[:, :, None]
    ok = (s > 0).expand_as(v)
    ratio = torch.where(ok, v.abs() / torch.where(s > 0, s, 1.0), 0.0)
    mags = torch.from_numpy(E2M1[:8])
    dist = (ratio[..., None] - mags).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best                       # one code, or two at a tie: the even one
    odd = torch.arange(8) % 2
    code = (near.double() * (2 - odd)).argmax(-1)
    code = torch.where(ok, code + 8 * (v < 0), 0).view(n, -1).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scale


def q4_values(codes, scale, k):
    """The values of a table, float64 [n, k]."""
    codes, scale = codes.cpu(), scale.cpu()
    n = codes.shape[0]
    code = torch.stack([codes & 15, codes >> 4], 2).reshape(n, -1).long()
    v = torch.from_numpy(E2M1)[code].view(n, -1, 32) * scale.double()[:, :, None]
    return v.reshape(n, -1)[:, :k]
