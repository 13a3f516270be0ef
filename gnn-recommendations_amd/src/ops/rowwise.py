"""Row-wise operators of the training path over libgnnrec: dropout from a counter-based
generator, layer norm, and the block between two hops that joins them.

    dropout(x, p, seed)                                  keep ? leaky(x) / (1 - p) : 0
    layer_norm(x, weight, bias)                          (x - mean) / sqrt(var + eps) w + b
    dropout_add_layer_norm(x, residual, weight, bias, p, seed)
                                                         h = residual + dropout(leaky(x)); LN(h), h

Tables on a ROCm device, fp32 / bf16 / fp16, 2-D row-major views with any row stride (0 too) or
contiguous tensors of any rank (rows are the last dimension); launched on torch's current stream
of the table's device. All differentiable (once, in reverse: a forward-mode tangent raises),
each backward pass one launch (two with a weight gradient) that repeats the forward's arithmetic
from its inputs: no mask, statistics or normalised rows are kept.

The dropout's mask: value (row, column) is dropped when its 16-bit draw is below
round(p * 65536), the others are scaled by 65536 / (65536 - round(p * 65536)). The draws are
Philox4x32-10 (Salmon et al., 2011) with key = `seed` and counter = (column // 8, row0 + row,
site), so they depend on nothing else: a row shard that passes its first global row as `row0`
draws what one device would, and a second dropout of the same step takes another `site`. `seed`
is an int or a one-element int64 tensor on the table's device; a captured graph reads the tensor
on every replay, so `seed.add_(1)` between replays (or captured in front) gives new masks.
A dropped value is 0 whatever x holds there, also an infinity or a NaN.

Nothing here can be traced into a graph of torch operators (torch.jit.trace, make_fx,
torch.export raise); under torch.compile a call runs between the compiled parts.

Forward and backward may be captured into a graph. As for any torch operator, no eager autograd
graph of the same leaves may be alive while a backward pass is captured.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.fx import _symbolic_trace as _fx_trace

from . import _lib
from ._lib import check, ptr

MAX_NORM_WIDTH = 16384    # csrc/layer_norm.hip kNormMaxD

Seed = Union[int, torch.Tensor]


_ENTRIES: dict = {}
_current_device = torch.cuda.current_device
# torch.cuda.current_stream(i).cuda_stream without the objects around it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda i: torch.cuda.current_stream(i).cuda_stream)


_jit_tracing = torch._C._is_tracing
_modes = torch._C._len_torch_dispatch_stack
_transform = torch._C._functorch.peek_interpreter_stack


def _refuse_tracing(name: str) -> None:
    """Raise if a graph is being recorded or tensors are functionalize's wrappers, which have no
    address (and not under another mode or transform)."""
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    functionalize = torch._C._functorch.TransformType.Functionalize
    if _jit_tracing() or get_proxy_mode() is not None or any(
            t.key() == functionalize for t in torch._C._functorch.get_interpreter_stack() or ()):
        raise RuntimeError(f"{name}: cannot be traced; a recorded graph would hold the result's "
                           "allocation without the launch that fills it, and this call's sizes")


def launch(name: str, device: torch.device, *args) -> None:
    """Call a C entry on `device`'s current stream, whatever device is current; refused while
    torch.jit.trace or make_fx records. The calls of a small table cost the host more than the
    GPU, so nothing is looked up twice here."""
    if _jit_tracing() or _fx_trace._is_fx_tracing_flag or _modes() or _transform() is not None:
        _refuse_tracing(name)
    fn = _ENTRIES.get(name)
    if fn is None:
        fn = _ENTRIES[name] = getattr(_lib.lib(), name)
    i = device.index
    if _current_device() == i:
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        check(rc, name)


def rows_of(t: torch.Tensor, what: str) -> torch.Tensor:
    """t as the 2-D [rows, width] view that the kernels take; raises where there is none."""
    if not t.is_cuda:
        raise ValueError(f"{what}: needs a tensor on a ROCm device, got {t.device}")
    if t.dtype not in _lib.DTYPES:
        raise TypeError(f"{what}: expected float32, bfloat16 or float16, got {t.dtype}")
    if t.dim() == 0 or t.shape[-1] == 0:
        raise ValueError(f"{what}: expected rows of at least one value, got {tuple(t.shape)}")
    if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1):
        return t
    if t.is_contiguous():
        return t.view(-1, t.shape[-1])
    raise ValueError(f"{what}: expected a 2-D row-major table (stride(1) == 1) or a contiguous "
                     "tensor")


def _empty_rows(t: torch.Tensor) -> torch.Tensor:
    """An uninitialised contiguous tensor of t's shape and type."""
    if t.is_contiguous():
        return torch.empty_like(t)
    return torch.empty_like(t, memory_format=torch.contiguous_format)


@lru_cache(maxsize=256)
def _norm_work_floats(rows: int, d: int) -> int:
    return _lib.lib().gnnrec_layer_norm_work_floats(rows, d)


def _dense_rows(t: Optional[torch.Tensor]):
    """(tensor, row stride) in a backward pass, of an incoming gradient (which may have any
    layout: an expanded scalar) or of a saved tensor (which a saved-tensor hook may have laid
    out anew): a 2-D row-major one as it is, another as a contiguous tensor."""
    if t is None:
        return None, 0
    if t.dim() == 2 and t.stride(1) == 1:
        return t, t.stride(0)
    t = t.contiguous()
    return t, t.shape[-1]


def _same(what: str, x: torch.Tensor, t: torch.Tensor, name: str) -> None:
    if t.device != x.device:
        raise ValueError(f"{what}: {name} on {t.device}, x on {x.device}")
    if t.dtype != x.dtype:
        raise TypeError(f"{what}: {name} is {t.dtype}, x is {x.dtype}")
    if t.shape != x.shape:
        raise ValueError(f"{what}: {name} is {tuple(t.shape)}, x is {tuple(x.shape)}")


def _drop_args(what: str, x: torch.Tensor, p: float, seed: Seed, site: int, row0: int,
               negative_slope: float):
    """(seed tensor or None, (p, host seed), (site, row0, slope)), checked: the mask's arguments
    of the C entries, around the seed's address."""
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{what}: p must be between 0 and 1, got {p}")
    if not 0 <= int(site) < 2 ** 32:
        raise ValueError(f"{what}: site must be a 32-bit number, got {site}")
    if not 0 <= int(row0) <= 2 ** 62:
        raise ValueError(f"{what}: row0 must be between 0 and 2^62, got {row0}")
    tensor = None
    if isinstance(seed, torch.Tensor):
        if seed.numel() != 1 or seed.dtype != torch.int64:
            raise TypeError(f"{what}: a seed tensor holds one int64, got {seed.dtype} "
                            f"{tuple(seed.shape)}")
        if seed.device != x.device:
            raise ValueError(f"{what}: seed on {seed.device}, x on {x.device}")
        tensor, seed = seed, 0
    return (tensor, (p, int(seed) & (2 ** 64 - 1)),
            (int(site), int(row0), float(negative_slope)))


_NO_MASK = (None, (0.0, 0), (0, 0, 1.0))


def _tracked(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd has to see a call with these inputs (otherwise its bookkeeping is
    skipped): one is recorded, or a forward-mode level is open. There an input may carry a
    tangent, whether it requires a gradient or not, and autograd refuses it (no jvp)."""
    return (forward_ad._current_level >= 0
            or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def _once(backward):
    """once_differentiable(backward), without its cost where no second derivative is asked for.
    A gradient with a forward-mode tangent is refused: the launch would lose it."""
    guarded = once_differentiable(backward)

    def wrapped(ctx, *grads):
        if forward_ad._current_level >= 0:
            if any(g is not None and forward_ad.unpack_dual(g).tangent is not None for g in grads):
                raise NotImplementedError("the row-wise operators' backward passes have no "
                                          "forward-mode derivative")
        return (guarded if torch.is_grad_enabled() else backward)(ctx, *grads)
    return staticmethod(wrapped)


def _dropout_forward(x, ldx, rows, mask):
    seed_t, pre, post = mask
    y = _empty_rows(x)
    d = x.shape[-1]
    launch("gnnrec_dropout_forward", x.device, _lib.DTYPES[x.dtype], rows, d, x.data_ptr(), ldx,
           y.data_ptr(), d, *pre, ptr(seed_t), *post)
    return y


def _dropout_backward(x, dy, rows, mask):
    seed_t, pre, post = mask
    x, ldx = _dense_rows(x)
    dy, lddy = _dense_rows(dy)
    dx = _empty_rows(dy)
    d = dy.shape[-1]
    launch("gnnrec_dropout_backward", dy.device, _lib.DTYPES[dy.dtype], rows, d, ptr(x), ldx,
           dy.data_ptr(), lddy, dx.data_ptr(), d, *pre, ptr(seed_t), *post)
    return dx


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ldx, rows, mask):
        y = _dropout_forward(x, ldx, rows, mask)
        seed_t, pre, post = mask
        ctx.save_for_backward(x if post[2] != 1.0 else None, seed_t)
        ctx.cfg = (rows, pre, post)
        return y

    @_once
    def backward(ctx, dy):
        x, seed_t = ctx.saved_tensors
        rows, pre, post = ctx.cfg
        return _dropout_backward(x, dy, rows, (seed_t, pre, post)), None, None, None


def dropout(x: torch.Tensor, p: float, seed: Seed, *, site: int = 0, row0: int = 0,
            negative_slope: float = 1.0) -> torch.Tensor:
    """Dropout of LeakyReLU(x) (negative_slope 1: of x) with a mask that is never stored; see
    the module's text for the mask, `seed`, `site` and `row0`. p = 1 drops everything, p = 0
    nothing. p counts in steps of 1 / 65536, and the scale goes by the step used."""
    x2 = rows_of(x, "dropout")
    mask = _drop_args("dropout", x, p, seed, site, row0, negative_slope)
    call = _Dropout.apply if _tracked(x) else _dropout_forward
    return call(x, x2.stride(0), x2.shape[0], mask)


def _norm_forward(x, res, w, b, cfg):
    """(y, h) = (LN(h) w + b, h), h = residual + dropout(leaky(x)); h is None without `keep_h`
    (layer_norm alone: h is x)."""
    keep_h, rows, ldx, ldr, t, wt, eps, (seed_t, pre, post) = cfg
    y = _empty_rows(x)
    h = torch.empty_like(y) if keep_h else None
    d = x.shape[-1]
    launch("gnnrec_layer_norm_forward", x.device, t, wt, rows, d, x.data_ptr(), ldx, ptr(res), ldr,
           ptr(w), ptr(b), eps, *pre, ptr(seed_t), *post, y.data_ptr(), d, ptr(h), d)
    return y, h


class _NormBlock(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, res, w, b, cfg):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, res, w, cfg[7][0])
        ctx.cfg = cfg
        ctx.b_dtype = b.dtype if b is not None else None
        return _norm_forward(x, res, w, b, cfg)

    @_once
    def backward(ctx, dy, dh):
        x, res, w, seed_t = ctx.saved_tensors
        _, rows, _, _, t, wt, eps, (_, pre, post) = ctx.cfg
        need_x, need_r, need_w, need_b, _ = ctx.needs_input_grad
        if dy is None and dh is None:
            return None, None, None, None, None
        if dy is None:
            # only h was used: nothing passes through the norm, which a row may not have (a NaN
            # in it, a constant one without eps)
            dx = _dropout_backward(x, dh, rows, (seed_t, pre, post)) if need_x else None
            return (dx, dh if need_r else None, torch.zeros_like(w) if need_w else None,
                    x.new_zeros(x.shape[-1], dtype=ctx.b_dtype) if need_b else None, None)
        x, ldx = _dense_rows(x)
        res, ldr = _dense_rows(res)
        dy, lddy = _dense_rows(dy)
        dh, lddh = _dense_rows(dh)
        d = x.shape[-1]
        dx = _empty_rows(x) if need_x else None
        dres = _empty_rows(x) if need_r else None
        dw = torch.empty_like(w) if need_w else None
        db = x.new_empty(d, dtype=ctx.b_dtype) if need_b else None
        work = None
        if need_w or need_b:
            work = x.new_empty(_norm_work_floats(rows, d), dtype=torch.float32)
        launch("gnnrec_layer_norm_backward", x.device, t, wt, rows, d, x.data_ptr(), ldx, ptr(res),
               ldr, ptr(w), eps, *pre, ptr(seed_t), *post, dy.data_ptr(), lddy, ptr(dh), lddh,
               ptr(dx), d, ptr(dres), d, ptr(dw), ptr(db), ptr(work))
        return dx, dres, dw, db, None


def _norm_block(what, keep_h, x, res, w, b, eps, mask):
    ldx, rows = _norm_args(what, x, w, b, eps)
    ldr = 0
    if res is not None:
        _same(what, x, res, "residual")
        ldr = rows_of(res, what).stride(0)
    t = _lib.DTYPES[x.dtype]
    wt = t if w is None and b is None else _lib.DTYPES[(b if w is None else w).dtype]
    cfg = (keep_h, rows, ldx, ldr, t, wt, float(eps), mask)
    call = _NormBlock.apply if _tracked(x, res, w, b) else _norm_forward
    return call(x, res, w, b, cfg)


def _norm_args(what: str, x: torch.Tensor, weight, bias, eps: float):
    """(row stride, rows) of x, everything checked."""
    x2 = rows_of(x, what)
    rows, d = x2.shape
    if d > MAX_NORM_WIDTH:
        raise NotImplementedError(f"{what}: rows of {d} values, at most {MAX_NORM_WIDTH}")
    if not eps >= 0.0:
        raise ValueError(f"{what}: eps must not be negative, got {eps}")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.device != x.device:
            raise ValueError(f"{what}: {name} on {t.device}, x on {x.device}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"{what}: {name} is {t.dtype}, expected {x.dtype} or float32")
        if t.shape != (d,) or (d > 1 and t.stride(0) != 1):
            raise ValueError(f"{what}: {name} must be a dense vector of {d} values")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"{what}: weight is {weight.dtype}, bias is {bias.dtype}")
    return x2.stride(0), rows


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension (at most
    MAX_NORM_WIDTH values; var divides by their number). weight and bias: x's dtype or float32,
    either may be None. Gradients of x, weight and bias; the weight's and the bias's are summed
    over all rows in fp32 in a fixed order. Deviations are squared in fp32: a row whose squares
    add up to more than it holds (64 deviations of 2.4e18) comes out as the bias."""
    return _norm_block("layer_norm", False, x, None, weight, bias, eps, _NO_MASK)[0]


def dropout_add_layer_norm(x: torch.Tensor, residual: Optional[torch.Tensor],
                           weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                           p: float, seed: Seed, *, site: int = 0, row0: int = 0,
                           negative_slope: float = 1.0, eps: float = 1e-5
                           ) -> Tuple[torch.Tensor, torch.Tensor]:
    """One layer's block in one pass: h = residual + dropout(LeakyReLU(x)) and y = LN(h) weight
    + bias; returns (y, h). residual None: h = dropout(LeakyReLU(x)). The mask is dropout()'s for
    the same p, seed, site and row0; the norm is layer_norm()'s, of the unrounded h."""
    what = "dropout_add_layer_norm"
    mask = _drop_args(what, x, p, seed, site, row0, negative_slope)
    return _norm_block(what, True, x, residual, weight, bias, eps, mask)
