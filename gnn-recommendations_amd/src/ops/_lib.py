"""ctypes binding of libgnnrec.so (the C ABI declared in include/gnnrec.h).

The library is the ONLY compute path for tensors on a ROCm device: there is no eager or
CPU fallback behind these functions. If the shared object is missing or does not export
the expected ABI version, :func:`lib` raises :class:`NativeLibraryError`.

torch must be imported before the library is loaded so that libgnnrec resolves
``libamdhip64.so.7`` to the HIP runtime torch already mapped (one runtime, shared streams).
"""
from __future__ import annotations

import ctypes as C
import os
from pathlib import Path

import torch  # (load order: torch's HIP runtime first)

_PKG_ROOT = Path(__file__).resolve().parents[2]
LIB_PATH = Path(os.environ.get("GNNREC_LIB", _PKG_ROOT / "lib" / "libgnnrec.so"))
ABI_VERSION = 12

# gnnrec.h gnnrec_dtype
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# gnnrec.h epilogue flags
EPI_ACC_INIT = 1
EPI_ACC_ADD = 2
EPI_ACC_DIV = 4
EPI_NO_Y = 8
EPI_ACC_X = 16
# gnnrec.h CSR hop flags (gnnrec_spmm_csr_heavy_f32)
CSR_FORK = 1
CSR_LIGHT_LATENCY = 2
CSR_LIGHT_THROUGHPUT = 4
CSR_TWO_LAUNCHES = 8
# column-ordered hop plan layout (include/gnnrec.h GNNREC_TILED_*)
TILED_WAVES = 8
TILED_GROUPS = 8
TILED_STEPS = 8
TILED_CHUNK = 64
TILED_TAIL = 8
TILED_QUAD_TAIL = 16
TILED_MAX_ROWS = 1279
TILED_SYNC_WORDS = 256
TILED_SYNC_ERR_WORD = 1   # GNNREC_TILED_SYNC_ERR_WORD: a non-quad plan on a quad build
TILED_HDR_WORDS = 4
TILED_MAX_LDX = 1024
TILED_MAX_PANEL = 1 << 20
TILED_MAX_CLASSES = 256
TILED_MAX_ROWS_FACTORED = 1232

_p = C.c_void_p
_u32 = C.c_uint32
_u64 = C.c_uint64
_f64 = C.c_double
_i64 = C.c_int64
_i32 = C.c_int32
_f32 = C.c_float

# name -> argtypes (all return int status unless listed in _RESTYPES)
_SIGNATURES = {
    "gnnrec_version": [],
    "gnnrec_abi_version": [],
    "gnnrec_last_error": [],
    "gnnrec_spmm_csr_f32": [_p, _p, _p, _i64, _p, _i64, _p, _i64, _i32, _i32, _p, _i64, _p,
                            _i64, _f32, _p],
    "gnnrec_lightgcn_f32": [_p, _p, _p, _i64, _p, _i32, _i32, _p, _p, _p, _p, _i64, _p],
    "gnnrec_spmm_csr_split_f32": [_p, _p, _p, _i64, _p, _i64, _p, _i64, _i32, _i32, _p, _i64,
                                  _p, _i64, _f32, _p, _i64, _i64, _p],
    "gnnrec_spmm_csr_masked_f32": [_p, _p, _p, _i64, _p, _i64, _p, _p, _p, _i64, _i32, _i32,
                                   _p, _i64, _p, _i64, _f32, _p, _i64, _i64, _p],
    "gnnrec_spmm_csr_heavy_f32": [_p, _p, _p, _i64, _p, _i64, _p, _p, _p, _i64, _i32, _i32,
                                  _p, _i64, _p, _i64, _f32, _p, _i64, _i64, _i64, _i32, _p],
    "gnnrec_lightgcn_heavy_f32": [_p, _p, _p, _i64, _p, _i32, _i32, _p, _p, _p, _p, _i64, _p,
                                  _i64, _i64, _i64, _i32, _p],
    "gnnrec_mark_active_rows": [_p, _p, _i64, _p, _i64, _p, _p],
    "gnnrec_tiled_plan_build": [_p, _p, _p, _i64, _i32, _i32, _i32, _i32, _p, _p, _p],
    "gnnrec_tiled_plan_emit": [_p, _p, _p, _p, _p, _p],
    "gnnrec_tiled_plan_free": [_p],
    "gnnrec_tiled_plan_device_scratch_words": [_i64, _i32],
    "gnnrec_csr_row_stats": [_p, _i64, _i64, _p, _p],
    "gnnrec_tiled_plan_device": [_p, _p, _p, _i64, _i32, _i32, _i32, _i64, _p, _i32, _p, _p, _p,
                                 _p, _p, _p, _p, _p],
    "gnnrec_spmm_tiled_supported": [_i32, _i32],
    "gnnrec_tiled_plan_quad": [],
    "gnnrec_tiled_plan_quad_offsets": [_p, _i64, _p, _p],
    "gnnrec_tiled_plan_quad_layout": [_p, _p, _i64, _i64, _i32, _p, _p, _p, _p, _p, _p, _p, _p,
                                      _p],
    "gnnrec_tiled_plan_factor": [_p, _p, _p, _p, _i64, _i32, _i64, _i64, _p, _p, _p, _i32, _p,
                                 _p, _p],
    "gnnrec_spmm_tiled_f32": [_p, _p, _p, _p, _p, _i32, _p, _p, _p, _i64, _i32, _p, _i64, _i64,
                              _p, _i64,
                              _i64, _i32, _i32, _p, _i64, _p, _i64, _f32, _p, _i64, _p, _i32, _p],
    "gnnrec_row_nonzero_f32": [_p, _i64, _i64, _i32, _p, _p],
    "gnnrec_spmm_sparse_src_f32": [_p, _p, _p, _i64, _i64, _p, _i64, _i64, _p, _i64, _p, _i64,
                                   _i32, _p, _p, _p],
    "gnnrec_lightgcn_split_f32": [_p, _p, _p, _i64, _p, _i32, _i32, _p, _p, _p, _p, _i64, _p,
                                  _i64, _i64, _p],
    "gnnrec_gas_f32": [_p, _i64, _i64, _i32, _i32, _p, _p, _p, _i64, _p],
    "gnnrec_spmm_gas_f32": [_p, _p, _p, _i64, _p, _i64, _p, _i64, _i32, _i32, _p, _p, _p],
    "gnnrec_spmm_ngcf_f32": [_p, _p, _p, _i64, _p, _i64, _p, _i64, _p, _i64, _i32, _p, _p, _p,
                             _p, _f32, _p, _p, _i32, _p, _p],
    "gnnrec_spmm_dense_f32": [_p, _p, _p, _i64, _p, _i64, _p, _i64, _i32, _p, _f32, _p, _i64,
                              _f32, _p, _i64, _i32, _f32, _f32, _p, _p],
    "gnnrec_ngcf_transform_f32": [_i64, _p, _i64, _p, _i64, _p, _i64, _i32, _p, _p, _p, _p,
                                  _f32, _p, _p, _i32, _p],
    "gnnrec_dense_transform_f32": [_i64, _p, _i64, _p, _i64, _i32, _p, _f32, _p, _i64, _f32,
                                   _p, _i64, _i32, _f32, _f32, _p],
    "gnnrec_rows_gemm_f32": [_i64, _p, _i64, _i32, _p, _i32, _p, _i64, _i32, _i32, _p, _i64,
                             _p, _i64, _f32, _p],
    "gnnrec_gat_aggregate_f32": [_p, _p, _i64, _p, _i64, _i64, _p, _p, _i64, _i64, _i32, _i32,
                                 _f32, _i32, _i32, _p, _i64, _i32, _p, _i64, _p, _i64, _f32, _i64,
                                 _p],
    "gnnrec_gat_heavy_f32": [_p, _p, _p, _p, _i64, _p, _p, _i64, _p, _p, _i64, _i64, _p, _p,
                             _i64, _i64, _i32, _i32, _f32, _i32, _i32, _p, _i64, _i32, _p, _i64,
                             _p, _i64, _f32, _p],
    "gnnrec_gat_aggregate_att_f32": [_p, _p, _i64, _p, _i64, _i64, _p, _i64, _p, _i32, _i32,
                                     _f32, _i32, _i32, _p, _i64, _i32, _p, _i64, _p, _i64, _f32,
                                     _i64, _p],
    "gnnrec_gat_heavy_att_f32": [_p, _p, _p, _p, _i64, _p, _p, _i64, _p, _p, _i64, _i64, _p,
                                 _i64, _p, _i32, _i32, _f32, _i32, _i32, _p, _i64, _i32, _p, _i64,
                                 _p, _i64, _f32, _p, _i32, _p],
    "gnnrec_gat_train_forward_f32": [_p, _p, _i64, _p, _i64, _p, _p, _i64, _i32, _i32, _f32,
                                     _f32, C.c_uint32, _p, _i64, _p],
    "gnnrec_gat_train_backward_f32": [_p, _p, _i64, _p, _i64, _p, _p, _i64, _i32, _i32, _f32,
                                      _f32, C.c_uint32, _p, _i64, _p, _i64, _p, _p, _i64, _p, _p,
                                      _p],
    "gnnrec_gat_train_forward_split_f32": [_p, _p, _i64, _p, _i64, _p, _p, _i64, _i32, _i32,
                                           _f32, _f32, C.c_uint32, _p, _i64, _p, _i64, _p, _p,
                                           _p, _i64, _p, _p, _i64, _p, _p],
    "gnnrec_gat_train_backward_split_f32": [_p, _p, _i64, _p, _i64, _p, _p, _i64, _i32, _i32,
                                            _f32, _f32, C.c_uint32, _p, _i64, _p, _i64, _p, _p,
                                            _i64, _p, _p, _i64, _p, _p, _p, _i64, _p, _p, _i64,
                                            _p, _p],
    "gnnrec_score_topk_f32": [_p, _i64, _i64, _p, _i64, _i64, _i32, _p, _p, _i32, _p, _p, _p],
    "gnnrec_score_topk_split_f32": [_p, _i64, _i64, _p, _i64, _i64, _i32, _p, _p, _i32, _i32,
                                    _p, _p, _p, _p, _p],
    "gnnrec_build_bipartite_csr": [_p, _p, _i64, _i64, _i64, _i32, _p, _p, _p, _p, _p, _i32],
    "gnnrec_normalize_values": [_p, _p, _p, _i64, _p, _i32, _p, _i32],
    "gnnrec_build_bipartite_csr_device": [_p, _p, _i64, _i64, _i64, _i32, _p, _p, _p, _p, _p,
                                          _p, _p, _p],
    "gnnrec_normalize_values_device": [_p, _p, _p, _i64, _p, _i32, _p, _p],
    "gnnrec_adam_step_f32": [_p, _p, _p, _p, _i64, _f32, C.c_double, C.c_double, _f32, _f32,
                             _f32, _p, _p],
    "gnnrec_dropout_forward": [_i32, _i64, _i64, _p, _i64, _p, _i64, _f64, _u64, _p, _u32, _i64,
                               _f32, _p],
    "gnnrec_dropout_backward": [_i32, _i64, _i64, _p, _i64, _p, _i64, _p, _i64, _f64, _u64, _p,
                                _u32, _i64, _f32, _p],
    "gnnrec_layer_norm_forward": [_i32, _i32, _i64, _i64, _p, _i64, _p, _i64, _p, _p, _f32, _f64,
                                  _u64, _p, _u32, _i64, _f32, _p, _i64, _p, _i64, _p],
    "gnnrec_layer_norm_work_floats": [_i64, _i64],
    "gnnrec_layer_norm_backward": [_i32, _i32, _i64, _i64, _p, _i64, _p, _i64, _p, _f32, _f64,
                                   _u64, _p, _u32, _i64, _f32, _p, _i64, _p, _i64, _p, _i64, _p,
                                   _i64, _p, _p, _p, _p],
    "gnnrec_quantize_q4": [_i32, _i64, _i64, _p, _i64, _p, _p, _p],
    "gnnrec_dequantize_q4": [_i64, _i64, _p, _p, _p, _i64, _p],
    "gnnrec_q4_matmul_work_bytes": [_i32, _i64, _i64, _i64],
    "gnnrec_q4_matmul": [_i32, _i32, _i64, _p, _i64, _i64, _i64, _p, _p, _p, _i64, _p, _p],
}
_RESTYPES = {"gnnrec_version": C.c_char_p, "gnnrec_last_error": C.c_char_p,
             "gnnrec_abi_version": C.c_int,
             "gnnrec_layer_norm_work_floats": C.c_int64,
             "gnnrec_q4_matmul_work_bytes": C.c_int64, "gnnrec_tiled_plan_device_scratch_words": C.c_int64}

EXPORTED = tuple(_SIGNATURES)


class NativeLibraryError(RuntimeError):
    """libgnnrec.so is missing, stale, or a call into it failed."""


_LIB = None


def lib() -> C.CDLL:
    """Load (once) and return the bound library; raises NativeLibraryError if unusable."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not LIB_PATH.exists():
        raise NativeLibraryError(
            f"{LIB_PATH} not found: build it with `python gnn-recommendations_amd/build_native.py` "
            "(or __graft_entry__.build()). There is no fallback path.")
    try:
        handle = C.CDLL(str(LIB_PATH), mode=C.RTLD_GLOBAL)
    except OSError as e:
        raise NativeLibraryError(f"cannot load {LIB_PATH}: {e}") from e
    for name, argtypes in _SIGNATURES.items():
        try:
            fn = getattr(handle, name)
        except AttributeError as e:
            raise NativeLibraryError(f"{LIB_PATH} does not export {name}") from e
        fn.argtypes = argtypes
        fn.restype = _RESTYPES.get(name, C.c_int)
    abi = handle.gnnrec_abi_version()
    if abi != ABI_VERSION:
        raise NativeLibraryError(f"{LIB_PATH} has ABI {abi}, expected {ABI_VERSION}: rebuild it")
    _LIB = handle
    return handle


def check(rc: int, what: str) -> None:
    """Raise with the library's thread-local message when a call returned non-zero."""
    if rc != 0:
        msg = lib().gnnrec_last_error().decode(errors="replace")
        kind = {-1: ValueError, -3: NotImplementedError}.get(rc, NativeLibraryError)
        raise kind(f"{what} failed ({rc}): {msg}")


def ptr(t) -> int:
    """Device/host address of a tensor (0 for None)."""
    return 0 if t is None else t.data_ptr()


def stream_of(device: torch.device) -> int:
    """The current torch stream on `device` as a raw hipStream_t (int)."""
    return torch.cuda.current_stream(device).cuda_stream


def version() -> str:
    return lib().gnnrec_version().decode()
