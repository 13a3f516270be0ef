"""Item tables in 4 bits and the scores of a few users against them, over libgnnrec.

    table = quantize_q4(item_emb)          # a quarter byte-for-byte of bfloat16, 0.56 B a value
    scores = q4_matmul(user_rows, table)   # [m, n_items]

A Q4Table holds E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), two a byte with the
even column in the low half, rows padded to whole groups of 32 columns, and one bfloat16 scale
for each group of a row. One user's scores read the table once, so they take the time of its
bytes: an eighth of an fp32 table's, and a catalogue that fits the caches eight times later.
Serving only: the scores carry no gradient and no forward-mode tangent, whatever x does.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import ptr
from .rowwise import launch, rows_of

GROUP = 32     # columns that share a scale; the kernels' matrix step is as deep
SHORT_COLUMNS = 256     # up to here the users need no workspace (csrc/q4.hip plan_of)


class Q4Table:
    """codes uint8 [n, 16 * ceil(k / 32)], scale bfloat16 [n, ceil(k / 32)], k columns.
    `scale` may have fewer columns, one for each `group` columns (a multiple of 32): it is
    repeated here once. The tensors are kept, not copied; what the codes' padding holds does
    not matter."""

    __slots__ = ("codes", "scale", "k")

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor, k: int, group: int = GROUP):
        k, group = int(k), int(group)
        if k < 1 or group < GROUP or group % GROUP:
            raise ValueError(f"Q4Table: k = {k} columns in groups of {group} (a multiple of 32)")
        groups = -(-k // GROUP)
        if codes.dtype != torch.uint8 or scale.dtype != torch.bfloat16:
            raise TypeError(f"Q4Table: codes uint8 and scale bfloat16, got {codes.dtype} and "
                            f"{scale.dtype}")
        if codes.dim() != 2 or codes.shape[1] != groups * 16:
            raise ValueError(f"Q4Table: codes must be [n, {groups * 16}] for {k} columns, got "
                             f"{tuple(codes.shape)}")
        if scale.shape != (codes.shape[0], -(-k // group)):
            raise ValueError(f"Q4Table: scale must be [{codes.shape[0]}, {-(-k // group)}], got "
                             f"{tuple(scale.shape)}")
        if codes.device != scale.device:
            raise ValueError(f"Q4Table: codes on {codes.device}, scale on {scale.device}")
        if group != GROUP:
            scale = scale.repeat_interleave(group // GROUP, dim=1)[:, :groups]
        codes = codes.contiguous()
        if codes.data_ptr() % 16:           # the kernels load 16 bytes
            codes = codes.clone()
        self.codes, self.scale, self.k = codes, scale.contiguous(), k

    @property
    def shape(self) -> Tuple[int, int]:
        return self.codes.shape[0], self.k

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scale.numel()

    def to(self, device) -> "Q4Table":
        return Q4Table(self.codes.to(device), self.scale.to(device), self.k)

    def dequantize(self) -> torch.Tensor:
        """The values the codes stand for, fp32 [n, k]."""
        if self.device.type != "cuda":
            raise ValueError(f"Q4Table.dequantize: needs a table on a ROCm device, got "
                             f"{self.device}")
        out = torch.empty(self.shape, dtype=torch.float32, device=self.device)
        launch("gnnrec_dequantize_q4", self.device, *self.shape, ptr(self.codes),
               ptr(self.scale), ptr(out), self.k)
        return out

    def __repr__(self) -> str:
        return f"Q4Table({self.shape[0]} x {self.k}, {self.nbytes} bytes, {self.device})"


def quantize_q4(w: torch.Tensor) -> Q4Table:
    """The 4-bit table of w's rows (2-D, fp32 / bf16 / fp16): a group's scale is its largest
    magnitude / 6 in bfloat16, a value's code the nearest to value / scale (ties to the even
    code). A group that holds an infinity or a NaN gets a NaN scale, so its row scores NaN."""
    if w.dim() != 2:
        raise ValueError(f"quantize_q4: expected a 2-D table, got {tuple(w.shape)}")
    w = rows_of(w.detach(), "quantize_q4")
    n, k = w.shape
    groups = -(-k // GROUP)
    codes = torch.empty((n, groups * 16), dtype=torch.uint8, device=w.device)
    scale = torch.empty((n, groups), dtype=torch.bfloat16, device=w.device)
    launch("gnnrec_quantize_q4", w.device, _lib.DTYPES[w.dtype], n, k, ptr(w), w.stride(0),
           ptr(codes), ptr(scale))
    return Q4Table(codes, scale, k)


def q4_matmul(x: torch.Tensor, table: Q4Table,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """x [m, k] (or [k]) times the table's rows: scores [m, n] (or [n]) in out_dtype (default
    x's). The products are exact (a code times a scale is not rounded) and summed in fp32, a
    group's before its scale is applied: values of x up to 2^110 cannot overflow there, and fp32
    values keep all their bits down to 2^-110 (below that the matrix cores drop parts smaller
    than 2^-126). x: fp32 / bf16 / fp16 rows of any stride, at most 65535 of them. The scores
    carry no gradient."""
    if not isinstance(table, Q4Table):
        raise TypeError(f"q4_matmul: expected a Q4Table, got {type(table).__name__}")
    codes, k = table.codes, table.k
    if out_dtype is None:
        out_dtype = x.dtype
    if out_dtype not in _lib.DTYPES:
        raise TypeError(f"q4_matmul: out_dtype must be float32, bfloat16 or float16, got "
                        f"{out_dtype}")
    if x.dim() not in (1, 2) or x.shape[-1] != k:
        raise ValueError(f"q4_matmul: x is {tuple(x.shape)}, the table has {k} columns")
    device = x.device
    if device != codes.device:
        raise ValueError(f"q4_matmul: x on {device}, table on {codes.device}")
    x2 = rows_of(x, "q4_matmul")
    m, n = x2.shape[0], codes.shape[0]
    if m > 65535:
        raise NotImplementedError(f"q4_matmul: {m} rows of x, at most 65535")
    out = torch.empty((m, n) if x.dim() == 2 else (n,), dtype=out_dtype, device=device)
    t = _lib.DTYPES[x.dtype]
    work = None
    if k > SHORT_COLUMNS:
        nbytes = _lib.lib().gnnrec_q4_matmul_work_bytes(t, m, n, k)
        work = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    launch("gnnrec_q4_matmul", device, t, _lib.DTYPES[out_dtype], m, x2.data_ptr(),
           x2.stride(0), n, k, codes.data_ptr(), table.scale.data_ptr(), out.data_ptr(), n,
           ptr(work))
    return out
