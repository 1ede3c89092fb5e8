"""Python binding of the B200 SpMM engine's C ABI (include/spmm_c.h, lib/libspmm_b200.so).

ctypes only: device buffers are passed as raw pointers (torch tensors are accepted and must
live on the current CUDA device), host buffers as numpy arrays. There is no fallback: if the
shared library is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import struct
from dataclasses import dataclass
from pathlib import Path

import numpy as np

HERE = Path(__file__).resolve().parent
LIB_PATH = HERE / "lib" / "libspmm_b200.so"
CXX_LIB_PATH = HERE / "lib" / "libspmm.so"

OK = 0
ERR = {
    -1: "SPMM_ERR_INVALID_ARG", -2: "SPMM_ERR_MISALIGNED", -3: "SPMM_ERR_CUDA", -4: "SPMM_ERR_NCCL",
    -5: "SPMM_ERR_TIMEOUT", -6: "SPMM_ERR_UNSUPPORTED", -7: "SPMM_ERR_NO_MEMORY", -8: "SPMM_ERR_BAD_INDEX",
    -9: "SPMM_ERR_IO", -10: "SPMM_ERR_TOO_LARGE",
}
CSR_AUTO, CSR_ROWWARP, CSR_MERGE = 0, 1, 2
DTYPE_F16, DTYPE_BF16, DTYPE_F32 = 0, 1, 2
BACKEND_CSR, BACKEND_TC = 0, 1

# Every symbol include/spmm_c.h declares (checked by the CPU test suite).
EXPORTS = [
    "spmm_status_string", "spmm_version", "spmm_csr_host_alloc", "spmm_csr_host_free", "spmm_csr_from_coo_host",
    "spmm_generate_uniform_csr", "spmm_generate_uniform_csr_fast", "spmm_generate_dense", "spmm_csr_row_slice_host", "spmm_csr_read_binary",
    "spmm_csr_write_binary", "spmm_csr_validate_host", "spmm_csr_to_bsr16_host", "spmm_bsr_host_free",
    "spmm_bsr_compute_stats", "spmm_nnz_balanced_bounds", "spmm_csr_f32", "spmm_csr_f32_workspace_size",
    "spmm_csr_f32_ws", "spmm_csr_f32_chunk", "spmm_csr_f32_host", "spmm_convert_f32", "spmm_bsr16",
    "spmm_bsr16_algo", "spmm_device_error", "spmm_hybrid_default_threshold", "spmm_hybrid_choose",
    "spmm_backend_name", "spmm_hybrid_run", "spmm_gpu_count", "spmm_multigpu_run", "spmm_unified_run",
    "spmm_unified_run_ex", "spmm_bsr16_plan_create", "spmm_bsr16_plan_execute", "spmm_bsr16_plan_info",
    "spmm_bsr16_plan_destroy", "spmm_bsr16_plan_a_stride",
    "spmm_csr_f32_noalloc", "spmm_csr_to_bsr16_device_count", "spmm_csr_to_bsr16_device_fill",
    "spmm_csr_plan_create", "spmm_csr_plan_execute", "spmm_csr_plan_info", "spmm_csr_plan_destroy",
    "spmm_csr_plan_k_phases", "spmm_csr_plan_launches",
    "spmm_comm_unique_id", "spmm_comm_init", "spmm_comm_wrap", "spmm_comm_info", "spmm_comm_destroy",
    "spmm_rank_plan_create", "spmm_rank_plan_info", "spmm_rank_run", "spmm_rank_submit", "spmm_rank_wait",
    "spmm_rank_execute", "spmm_rank_gather_b",
    "spmm_rank_plan_buffers", "spmm_rank_plan_destroy",
    "spmm_route_workspace_size", "spmm_route_build", "spmm_route_gather", "spmm_route_combine",
    "spmm_route_combine_grad", "spmm_grouped_mm", "spmm_grouped_mm_dx", "spmm_grouped_mm_dw",
    "spmm_lora_workspace_size", "spmm_lora",
]


class SpmmError(RuntimeError):
    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {ERR.get(status, status)} ({status_string(status)})")


class CsrView(C.Structure):
    _fields_ = [("rows", C.c_int32), ("cols", C.c_int32), ("nnz", C.c_int32), ("row_ptr", C.c_void_p),
                ("col_idx", C.c_void_p), ("values", C.c_void_p)]


class CsrHost(C.Structure):
    _fields_ = [("rows", C.c_int32), ("cols", C.c_int32), ("nnz", C.c_int32), ("row_ptr", C.POINTER(C.c_int32)),
                ("col_idx", C.POINTER(C.c_int32)), ("values", C.POINTER(C.c_float))]


class BsrView(C.Structure):
    _fields_ = [("rows", C.c_int32), ("cols", C.c_int32), ("block_rows", C.c_int32), ("block_cols", C.c_int32),
                ("num_blocks", C.c_int32), ("nnz", C.c_int32), ("row_ptr", C.c_void_p), ("col_idx", C.c_void_p),
                ("values", C.c_void_p), ("dtype", C.c_int32)]


class BsrHost(C.Structure):
    _fields_ = [("rows", C.c_int32), ("cols", C.c_int32), ("block_rows", C.c_int32), ("block_cols", C.c_int32),
                ("num_blocks", C.c_int32), ("nnz", C.c_int32), ("dtype", C.c_int32),
                ("row_ptr", C.POINTER(C.c_int32)), ("col_idx", C.POINTER(C.c_int32)),
                ("values", C.POINTER(C.c_uint16))]


class BsrStats(C.Structure):
    _fields_ = [("num_blocks", C.c_int32), ("stored_elements", C.c_int64), ("original_nnz", C.c_int32),
                ("fill_in_ratio", C.c_double), ("block_density", C.c_double)]


class CsrTuning(C.Structure):
    _fields_ = [("chunk", C.c_int32), ("col_pass", C.c_int32), ("b_policy", C.c_int32), ("k_phases", C.c_int32),
                ("schedule", C.c_int32), ("phase_mode", C.c_int32), ("reserved", C.c_int32 * 2)]


class HybridPlan(C.Structure):
    _fields_ = [("backend", C.c_int32), ("fill_in_ratio", C.c_double), ("block_density", C.c_double),
                ("threshold", C.c_float), ("n_aligned", C.c_int32), ("reason", C.c_char_p)]


class RouteView(C.Structure):
    _fields_ = [("tokens", C.c_int32), ("topk", C.c_int32), ("rows", C.c_int32), ("pos", C.c_void_p)]


class LoraView(C.Structure):
    _fields_ = [("adapters", C.c_int32), ("rank", C.c_int32), ("N", C.c_int32), ("K", C.c_int32), ("dtype", C.c_int32),
                ("a", C.c_void_p), ("b", C.c_void_p), ("scale", C.c_void_p)]


_lib: C.CDLL | None = None


def lib() -> C.CDLL:
    """Load lib/libspmm_b200.so (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(f"{LIB_PATH} is missing: build it with `make -C {HERE}` (or __graft_entry__.build())")
    L = C.CDLL(str(LIB_PATH))
    vp, i32, i64, f32 = C.c_void_p, C.c_int32, C.c_int64, C.c_float
    sig = {
        "spmm_status_string": (C.c_char_p, [C.c_int]),
        "spmm_version": (C.c_int, []),
        "spmm_csr_host_alloc": (C.c_int, [i32, i32, i32, C.POINTER(CsrHost)]),
        "spmm_csr_host_free": (None, [C.POINTER(CsrHost)]),
        "spmm_csr_from_coo_host": (C.c_int, [i32, i32, i32, vp, vp, vp, C.POINTER(CsrHost)]),
        "spmm_generate_uniform_csr": (C.c_int, [i32, i32, f32, i32, C.POINTER(CsrHost)]),
        "spmm_generate_uniform_csr_fast": (C.c_int, [i32, i32, f32, C.c_int64, i32, C.POINTER(CsrHost)]),
        "spmm_generate_dense": (C.c_int, [i32, i32, i32, vp]),
        "spmm_csr_row_slice_host": (C.c_int, [C.POINTER(CsrView), i32, i32, C.POINTER(CsrHost)]),
        "spmm_csr_read_binary": (C.c_int, [C.c_char_p, C.POINTER(CsrHost)]),
        "spmm_csr_write_binary": (C.c_int, [C.POINTER(CsrView), C.c_char_p]),
        "spmm_csr_validate_host": (C.c_int, [C.POINTER(CsrView), C.POINTER(i32)]),
        "spmm_csr_to_bsr16_host": (C.c_int, [C.POINTER(CsrView), i32, C.POINTER(BsrHost)]),
        "spmm_bsr_host_free": (None, [C.POINTER(BsrHost)]),
        "spmm_bsr_compute_stats": (C.c_int, [C.POINTER(BsrView), C.POINTER(BsrStats)]),
        "spmm_nnz_balanced_bounds": (C.c_int, [vp, i32, i64, i32, vp]),
        "spmm_csr_f32": (C.c_int, [C.POINTER(CsrView), vp, vp, i32, i32, vp]),
        "spmm_csr_f32_workspace_size": (C.c_int, [C.POINTER(CsrView), i32, i32, C.POINTER(CsrTuning),
                                                   C.POINTER(C.c_size_t)]),
        "spmm_csr_f32_ws": (C.c_int, [C.POINTER(CsrView), vp, vp, i32, i32, C.POINTER(CsrTuning), vp, C.c_size_t,
                                      vp]),
        "spmm_csr_f32_chunk": (C.c_int, [C.POINTER(CsrView), i32, i32, C.POINTER(CsrTuning), C.POINTER(i32)]),
        "spmm_csr_f32_host": (C.c_int, [C.POINTER(CsrView), vp, vp, i32, i32, vp]),
        "spmm_convert_f32": (C.c_int, [vp, vp, i64, i32, vp]),
        "spmm_bsr16": (C.c_int, [C.POINTER(BsrView), vp, vp, i32, vp]),
        "spmm_bsr16_algo": (C.c_int, [C.POINTER(BsrView), vp, vp, i32, i32, vp]),
        "spmm_bsr16_plan_create": (C.c_int, [C.POINTER(BsrView), i32, vp, C.POINTER(vp)]),
        "spmm_bsr16_plan_execute": (C.c_int, [vp, vp, vp, vp]),
        "spmm_bsr16_plan_info": (C.c_int, [vp, C.POINTER(i32), C.POINTER(i32), C.POINTER(C.c_size_t)]),
        "spmm_bsr16_plan_destroy": (None, [vp]),
        "spmm_bsr16_plan_a_stride": (C.c_int, [vp, C.POINTER(i32)]),
        "spmm_device_error": (C.c_int, [i32, C.POINTER(i32), C.POINTER(i64), i32]),
        "spmm_hybrid_default_threshold": (f32, []),
        "spmm_hybrid_choose": (C.c_int, [C.POINTER(CsrView), i32, f32, C.POINTER(HybridPlan)]),
        "spmm_backend_name": (C.c_char_p, [i32]),
        "spmm_hybrid_run": (C.c_int, [C.POINTER(HybridPlan), C.POINTER(CsrView), vp, vp, i32, i32, i32,
                                      C.POINTER(f32)]),
        "spmm_gpu_count": (C.c_int, []),
        "spmm_multigpu_run": (C.c_int, [C.POINTER(CsrView), vp, vp, i32, i32, i32, i32, C.POINTER(f32),
                                        C.POINTER(i32), vp, vp, C.POINTER(f32)]),
        "spmm_unified_run": (C.c_int, [C.POINTER(CsrView), vp, vp, i32, i32, i32, C.POINTER(f32)]),
        "spmm_unified_run_ex": (C.c_int, [C.POINTER(CsrView), vp, vp, i32, C.c_size_t, i32, i32, C.POINTER(f32),
                                          C.POINTER(i32)]),
        "spmm_csr_f32_noalloc": (C.c_int, [C.POINTER(CsrView), vp, vp, i32, i32, vp]),
        "spmm_csr_to_bsr16_device_count": (C.c_int, [C.POINTER(CsrView), vp, C.POINTER(i32), vp]),
        "spmm_csr_to_bsr16_device_fill": (C.c_int, [C.POINTER(CsrView), vp, vp, vp, i32, vp]),
        "spmm_csr_plan_create": (C.c_int, [C.POINTER(CsrView), i32, C.POINTER(CsrTuning), vp, C.POINTER(vp)]),
        "spmm_csr_plan_execute": (C.c_int, [vp, vp, vp, vp]),
        "spmm_csr_plan_info": (C.c_int, [vp, C.POINTER(i32), C.POINTER(i32), C.POINTER(C.c_size_t)]),
        "spmm_csr_plan_k_phases": (C.c_int, [vp, C.POINTER(i32)]),
        "spmm_csr_plan_launches": (C.c_int, [vp, C.POINTER(i32)]),
        "spmm_csr_plan_destroy": (None, [vp]),
        "spmm_comm_unique_id": (C.c_int, [vp]),
        "spmm_comm_init": (C.c_int, [vp, i32, i32, i32, C.POINTER(vp)]),
        "spmm_comm_wrap": (C.c_int, [vp, i32, C.POINTER(vp)]),
        "spmm_comm_info": (C.c_int, [vp, C.POINTER(i32), C.POINTER(i32), C.POINTER(i32)]),
        "spmm_comm_destroy": (None, [vp]),
        "spmm_rank_plan_create": (C.c_int, [vp, C.POINTER(CsrView), i32, vp, C.POINTER(vp)]),
        "spmm_rank_plan_info": (C.c_int, [vp, C.POINTER(i32), C.POINTER(i32), C.POINTER(i32), C.POINTER(i32),
                                          C.POINTER(i32), C.POINTER(i32), C.POINTER(i32)]),
        "spmm_rank_run": (C.c_int, [vp, C.POINTER(CsrView), vp, vp, vp]),
        "spmm_rank_submit": (C.c_int, [vp, C.POINTER(CsrView), vp, vp, vp]),
        "spmm_rank_wait": (C.c_int, [vp, vp]),
        "spmm_rank_execute": (C.c_int, [vp, vp]),
        "spmm_rank_gather_b": (C.c_int, [vp, vp]),
        "spmm_rank_plan_buffers": (C.c_int, [vp, C.POINTER(vp), C.POINTER(vp)]),
        "spmm_rank_plan_destroy": (None, [vp]),
        "spmm_route_workspace_size": (C.c_int, [i32, i32, i32, C.POINTER(C.c_size_t)]),
        "spmm_route_build": (C.c_int, [vp, i32, i32, i32, vp, vp, vp, vp, C.c_size_t, vp]),
        "spmm_route_gather": (C.c_int, [vp, vp, i64, vp, i64, i32, i32, vp]),
        "spmm_route_combine": (C.c_int, [vp, vp, i64, vp, vp, i64, i32, i32, vp]),
        "spmm_route_combine_grad": (C.c_int, [vp, vp, i64, vp, i64, vp, vp, i64, vp, i32, i32, vp]),
        "spmm_grouped_mm": (C.c_int, [vp, i32, i32, vp, i64, vp, vp, i64, i32, i32, i32, i32, vp]),
        "spmm_grouped_mm_dx": (C.c_int, [vp, i32, i32, vp, i64, vp, vp, i64, i32, i32, i32, i32, vp]),
        "spmm_grouped_mm_dw": (C.c_int, [vp, i32, i32, vp, i64, vp, i64, vp, i32, i32, i32, i32, vp]),
        "spmm_lora_workspace_size": (C.c_int, [C.POINTER(LoraView), i32, i32, C.POINTER(C.c_size_t)]),
        "spmm_lora": (C.c_int, [vp, vp, vp, i32, i32, vp, i64, vp, i64, vp, i64, vp, C.c_size_t, vp]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(L, name)
        fn.restype = res
        fn.argtypes = args
    _lib = L
    return L


def status_string(status: int) -> str:
    try:
        return lib().spmm_status_string(status).decode()
    except Exception:  # noqa: BLE001 - used while formatting another error
        return "?"


def check(status: int, what: str) -> None:
    if status != OK:
        raise SpmmError(status, what)


# ------------------------------------------------------------------ pointers


def ptr(x) -> int:
    """Raw address of a torch tensor or numpy array (0 for None)."""
    if x is None:
        return 0
    if hasattr(x, "data_ptr"):
        return int(x.data_ptr())
    return int(x.ctypes.data)


def stream_ptr(stream) -> int:
    if stream is None:
        return 0
    if hasattr(stream, "cuda_stream"):
        return int(stream.cuda_stream)
    return int(stream)


# ------------------------------------------------------------------ host CSR


@dataclass
class HostCSR:
    rows: int
    cols: int
    row_ptr: np.ndarray
    col_idx: np.ndarray
    values: np.ndarray

    @property
    def nnz(self) -> int:
        return int(self.col_idx.size)

    def view(self) -> CsrView:
        return CsrView(self.rows, self.cols, self.nnz, ptr(self.row_ptr), ptr(self.col_idx), ptr(self.values))


def _adopt(h: CsrHost) -> HostCSR:
    L = lib()
    rp = np.ctypeslib.as_array(h.row_ptr, shape=(h.rows + 1,)).copy()
    ci = np.ctypeslib.as_array(h.col_idx, shape=(h.nnz,)).copy() if h.nnz else np.zeros(0, np.int32)
    v = np.ctypeslib.as_array(h.values, shape=(h.nnz,)).copy() if h.nnz else np.zeros(0, np.float32)
    out = HostCSR(h.rows, h.cols, rp, ci, v)
    L.spmm_csr_host_free(C.byref(h))
    return out


def generate_uniform_csr(rows: int, cols: int, density: float, seed: int) -> HostCSR:
    h = CsrHost()
    check(lib().spmm_generate_uniform_csr(rows, cols, density, seed, C.byref(h)), "spmm_generate_uniform_csr")
    return _adopt(h)


def generate_uniform_csr_fast(rows: int, cols: int, density: float, seed: int, threads: int = 0) -> HostCSR:
    """Geometric-gap uniform CSR (not the reference's mt19937 stream; same expected nnz)."""
    h = CsrHost()
    check(lib().spmm_generate_uniform_csr_fast(rows, cols, density, seed, threads, C.byref(h)),
          "spmm_generate_uniform_csr_fast")
    return _adopt(h)


def generate_dense(rows: int, cols: int, seed: int) -> np.ndarray:
    out = np.empty((rows, cols), dtype=np.float32)
    check(lib().spmm_generate_dense(rows, cols, seed, ptr(out)), "spmm_generate_dense")
    return out


def csr_from_coo(rows: int, cols: int, r, c, v) -> HostCSR:
    r = np.ascontiguousarray(r, np.int32)
    c = np.ascontiguousarray(c, np.int32)
    v = np.ascontiguousarray(v, np.float32)
    h = CsrHost()
    check(lib().spmm_csr_from_coo_host(rows, cols, int(v.size), ptr(r), ptr(c), ptr(v), C.byref(h)),
          "spmm_csr_from_coo_host")
    return _adopt(h)


def row_slice(A: HostCSR, b: int, e: int) -> HostCSR:
    h = CsrHost()
    v = A.view()
    check(lib().spmm_csr_row_slice_host(C.byref(v), b, e, C.byref(h)), "spmm_csr_row_slice_host")
    return _adopt(h)


def read_binary(path: str | os.PathLike) -> HostCSR:
    h = CsrHost()
    check(lib().spmm_csr_read_binary(os.fsencode(path), C.byref(h)), "spmm_csr_read_binary")
    return _adopt(h)


def write_binary(A: HostCSR, path: str | os.PathLike) -> None:
    v = A.view()
    check(lib().spmm_csr_write_binary(C.byref(v), os.fsencode(path)), "spmm_csr_write_binary")


def validate(A: HostCSR) -> int:
    """-1 when A is well formed, else the first bad row (raises on bad arguments)."""
    bad = C.c_int32(-1)
    v = A.view()
    rc = lib().spmm_csr_validate_host(C.byref(v), C.byref(bad))
    if rc == OK:
        return -1
    if bad.value >= 0:
        return bad.value
    raise SpmmError(rc, "spmm_csr_validate_host")


@dataclass
class HostBSR:
    rows: int
    cols: int
    block_rows: int
    block_cols: int
    row_ptr: np.ndarray
    col_idx: np.ndarray
    values: np.ndarray  # uint16 bits
    nnz: int
    dtype: int

    @property
    def num_blocks(self) -> int:
        return int(self.col_idx.size)

    def view(self) -> BsrView:
        return BsrView(self.rows, self.cols, self.block_rows, self.block_cols, self.num_blocks, self.nnz,
                       ptr(self.row_ptr), ptr(self.col_idx), ptr(self.values), self.dtype)


def csr_to_bsr16(A: HostCSR, dtype: int = DTYPE_F16) -> HostBSR:
    b = BsrHost()
    v = A.view()
    check(lib().spmm_csr_to_bsr16_host(C.byref(v), dtype, C.byref(b)), "spmm_csr_to_bsr16_host")
    nb = b.num_blocks
    out = HostBSR(b.rows, b.cols, b.block_rows, b.block_cols,
                  np.ctypeslib.as_array(b.row_ptr, shape=(b.block_rows + 1,)).copy(),
                  np.ctypeslib.as_array(b.col_idx, shape=(nb,)).copy() if nb else np.zeros(0, np.int32),
                  np.ctypeslib.as_array(b.values, shape=(nb * 256,)).copy() if nb else np.zeros(0, np.uint16),
                  b.nnz, b.dtype)
    lib().spmm_bsr_host_free(C.byref(b))
    return out


def bsr_stats(B: HostBSR) -> dict:
    s = BsrStats()
    v = B.view()
    check(lib().spmm_bsr_compute_stats(C.byref(v), C.byref(s)), "spmm_bsr_compute_stats")
    return {"num_blocks": s.num_blocks, "stored_elements": s.stored_elements, "original_nnz": s.original_nnz,
            "fill_in_ratio": s.fill_in_ratio, "block_density": s.block_density}


def nnz_balanced_bounds(row_ptr: np.ndarray, rows: int, nnz: int, G: int) -> np.ndarray:
    row_ptr = np.ascontiguousarray(row_ptr, np.int32)
    out = np.zeros(G + 1, dtype=np.int32)
    check(lib().spmm_nnz_balanced_bounds(ptr(row_ptr), rows, nnz, G, ptr(out)), "spmm_nnz_balanced_bounds")
    return out


def hybrid_choose(A: HostCSR, N: int, threshold: float = 0.0) -> dict:
    p = HybridPlan()
    v = A.view()
    check(lib().spmm_hybrid_choose(C.byref(v), N, threshold, C.byref(p)), "spmm_hybrid_choose")
    return {"backend": p.backend, "backend_name": lib().spmm_backend_name(p.backend).decode(),
            "fill_in_ratio": p.fill_in_ratio, "block_density": p.block_density, "threshold": p.threshold,
            "n_aligned": bool(p.n_aligned), "reason": p.reason.decode(), "_plan": p}


# ------------------------------------------------------------------ device compute


def device_view(rows: int, cols: int, row_ptr, col_idx, values) -> CsrView:
    """CsrView over device tensors (int32 row_ptr/col_idx, float32 values)."""
    nnz = int(col_idx.numel()) if hasattr(col_idx, "numel") else int(col_idx.size)
    return CsrView(rows, cols, nnz, ptr(row_ptr), ptr(col_idx), ptr(values))


def csr_f32(A: CsrView, B, Cout, N: int, algo: int = CSR_AUTO, stream=None) -> None:
    check(lib().spmm_csr_f32(C.byref(A), ptr(B), ptr(Cout), N, algo, stream_ptr(stream)), "spmm_csr_f32")


def csr_f32_ws(A: CsrView, B, Cout, N: int, algo: int, tuning: CsrTuning | None, ws, ws_bytes: int,
               stream=None) -> None:
    t = C.byref(tuning) if tuning is not None else None
    check(lib().spmm_csr_f32_ws(C.byref(A), ptr(B), ptr(Cout), N, algo, t, ptr(ws), ws_bytes, stream_ptr(stream)),
          "spmm_csr_f32_ws")


def csr_workspace_size(A: CsrView, N: int, algo: int = CSR_AUTO, tuning: CsrTuning | None = None) -> int:
    n = C.c_size_t()
    t = C.byref(tuning) if tuning is not None else None
    check(lib().spmm_csr_f32_workspace_size(C.byref(A), N, algo, t, C.byref(n)), "spmm_csr_f32_workspace_size")
    return int(n.value)


def csr_chunk(A: CsrView, N: int, algo: int = CSR_AUTO, tuning: CsrTuning | None = None) -> int:
    c = C.c_int32()
    t = C.byref(tuning) if tuning is not None else None
    check(lib().spmm_csr_f32_chunk(C.byref(A), N, algo, t, C.byref(c)), "spmm_csr_f32_chunk")
    return int(c.value)


def csr_f32_host(A: HostCSR, B: np.ndarray, Cout: np.ndarray, N: int, algo: int = CSR_AUTO, stream=None) -> None:
    v = A.view()
    check(lib().spmm_csr_f32_host(C.byref(v), ptr(B), ptr(Cout), N, algo, stream_ptr(stream)), "spmm_csr_f32_host")


def convert_f32(src, dst, n: int, dtype: int = DTYPE_F16, stream=None) -> None:
    check(lib().spmm_convert_f32(ptr(src), ptr(dst), n, dtype, stream_ptr(stream)), "spmm_convert_f32")


def bsr16(A: BsrView, B16, Cout, N: int, algo: int = 0, stream=None) -> None:
    check(lib().spmm_bsr16_algo(C.byref(A), ptr(B16), ptr(Cout), N, algo, stream_ptr(stream)), "spmm_bsr16")


class BsrPlan:
    """spmm_bsr16_plan_* wrapper: precompute the per-CTA schedule once, execute many times."""

    def __init__(self, A: BsrView, N: int, stream=None):
        self._A = A
        self.N = N
        h = C.c_void_p()
        check(lib().spmm_bsr16_plan_create(C.byref(A), N, stream_ptr(stream), C.byref(h)), "spmm_bsr16_plan_create")
        self._h = h
        g, ms, nb = C.c_int32(), C.c_int32(), C.c_size_t()
        check(lib().spmm_bsr16_plan_info(h, C.byref(g), C.byref(ms), C.byref(nb)), "spmm_bsr16_plan_info")
        self.group, self.max_steps, self.schedule_bytes = int(g.value), int(ms.value), int(nb.value)
        st = C.c_int32()
        check(lib().spmm_bsr16_plan_a_stride(h, C.byref(st)), "spmm_bsr16_plan_a_stride")
        self.a_stride = int(st.value)  # block stride of the grouped A copies (0: none)

    def execute(self, B16, Cout, stream=None) -> None:
        check(lib().spmm_bsr16_plan_execute(self._h, ptr(B16), ptr(Cout), stream_ptr(stream)), "spmm_bsr16_plan_execute")

    def close(self) -> None:
        if self._h:
            lib().spmm_bsr16_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


class CsrPlan:
    """spmm_csr_plan_* wrapper: inspect A once, execute many times (no allocation per call)."""

    def __init__(self, A: CsrView, N: int, tuning: CsrTuning | None = None, stream=None):
        self._A = A  # keep the view alive: the plan refers to the same device arrays
        self.N = N
        h = C.c_void_p()
        t = C.byref(tuning) if tuning is not None else None
        check(lib().spmm_csr_plan_create(C.byref(A), N, t, stream_ptr(stream), C.byref(h)), "spmm_csr_plan_create")
        self._h = h
        algo, mx, ws = C.c_int32(), C.c_int32(), C.c_size_t()
        check(lib().spmm_csr_plan_info(h, C.byref(algo), C.byref(mx), C.byref(ws)), "spmm_csr_plan_info")
        self.algo, self.max_row, self.ws_bytes = int(algo.value), int(mx.value), int(ws.value)
        ph = C.c_int32()
        check(lib().spmm_csr_plan_k_phases(h, C.byref(ph)), "spmm_csr_plan_k_phases")
        self.k_phases = int(ph.value)  # column phases
        check(lib().spmm_csr_plan_launches(h, C.byref(ph)), "spmm_csr_plan_launches")
        self.launches = int(ph.value)  # kernel launches per execute

    def execute(self, B, Cout, stream=None) -> None:
        check(lib().spmm_csr_plan_execute(self._h, ptr(B), ptr(Cout), stream_ptr(stream)), "spmm_csr_plan_execute")

    def close(self) -> None:
        if self._h:
            lib().spmm_csr_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


def csr_to_bsr16_device(A: CsrView, dtype: int = DTYPE_F16, stream=None):
    """CSR (device view) -> BSR-16 on the GPU. Returns (BsrView, [row_ptr, col_idx, values]
    torch tensors that own the memory)."""
    import torch

    br = (A.rows + 15) // 16
    rp = torch.empty(br + 1, dtype=torch.int32, device="cuda")
    nb = C.c_int32()
    check(lib().spmm_csr_to_bsr16_device_count(C.byref(A), ptr(rp), C.byref(nb), stream_ptr(stream)),
          "spmm_csr_to_bsr16_device_count")
    n = int(nb.value)
    ci = torch.empty(max(n, 1), dtype=torch.int32, device="cuda")
    vals = torch.empty(max(n * 256, 2), dtype=torch.int16, device="cuda")
    check(lib().spmm_csr_to_bsr16_device_fill(C.byref(A), ptr(rp), ptr(ci), ptr(vals), dtype, stream_ptr(stream)),
          "spmm_csr_to_bsr16_device_fill")
    view = BsrView(A.rows, A.cols, br, (A.cols + 15) // 16, n, A.nnz, ptr(rp), ptr(ci), ptr(vals), dtype)
    return view, [rp, ci, vals]


def device_error(device: int = 0, clear: bool = True) -> tuple[int, int]:
    code, detail = C.c_int32(), C.c_int64()
    check(lib().spmm_device_error(device, C.byref(code), C.byref(detail), int(clear)), "spmm_device_error")
    return int(code.value), int(detail.value)


def gpu_count() -> int:
    return int(lib().spmm_gpu_count())


def hybrid_run(plan: dict, A: HostCSR, B: np.ndarray, Cout: np.ndarray, N: int, warmup: int, iters: int) -> float:
    ms = C.c_float()
    v = A.view()
    check(lib().spmm_hybrid_run(C.byref(plan["_plan"]), C.byref(v), ptr(B), ptr(Cout), N, warmup, iters,
                                C.byref(ms)), "spmm_hybrid_run")
    return float(ms.value)


def multigpu_run(A: HostCSR, B: np.ndarray, Cout: np.ndarray, N: int, gpus: int, warmup: int, iters: int) -> dict:
    ms, used, bc = C.c_float(), C.c_int32(), C.c_float()
    rows = np.zeros(max(gpus, 1), np.int32)
    nnz = np.zeros(max(gpus, 1), np.int32)
    v = A.view()
    check(lib().spmm_multigpu_run(C.byref(v), ptr(B), ptr(Cout), N, gpus, warmup, iters, C.byref(ms), C.byref(used),
                                  ptr(rows), ptr(nnz), C.byref(bc)), "spmm_multigpu_run")
    g = int(used.value)
    return {"time_ms": float(ms.value), "num_gpus": g, "rows": rows[:g].tolist(), "nnz": nnz[:g].tolist(),
            "bcast_ms": float(bc.value)}


def unified_run(A: HostCSR, B: np.ndarray, Cout: np.ndarray, N: int, warmup: int, iters: int) -> float:
    ms = C.c_float()
    v = A.view()
    check(lib().spmm_unified_run(C.byref(v), ptr(B), ptr(Cout), N, warmup, iters, C.byref(ms)), "spmm_unified_run")
    return float(ms.value)


def unified_run_ex(A: HostCSR, B: np.ndarray, Cout: np.ndarray, N: int, device_budget: int, warmup: int,
                   iters: int) -> tuple[float, int]:
    """spmm_unified_run_ex: (median ms per pass, column phases used)."""
    ms, ph = C.c_float(), C.c_int32()
    v = A.view()
    check(lib().spmm_unified_run_ex(C.byref(v), ptr(B), ptr(Cout), N, device_budget, warmup, iters, C.byref(ms),
                                    C.byref(ph)), "spmm_unified_run_ex")
    return float(ms.value), int(ph.value)


# ------------------------------------------------------------------ multi-GPU, one process per GPU

COMM_ID_BYTES = 128


def comm_unique_id() -> bytes:
    """A fresh communicator id (spmm_comm_unique_id): make it on one rank, send the bytes to all."""
    buf = (C.c_uint8 * COMM_ID_BYTES)()
    check(lib().spmm_comm_unique_id(buf), "spmm_comm_unique_id")
    return bytes(buf)


class RankComm:
    """spmm_comm_*: this process's member of an NCCL communicator over `world` ranks (one GPU each;
    the current device is this rank's)."""

    def __init__(self, comm_id: bytes, world: int, rank: int, timeout_ms: int = 0):
        if len(comm_id) != COMM_ID_BYTES:
            raise ValueError("communicator id must be 128 bytes")
        buf = (C.c_uint8 * COMM_ID_BYTES).from_buffer_copy(comm_id)
        h = C.c_void_p()
        check(lib().spmm_comm_init(buf, world, rank, timeout_ms, C.byref(h)), "spmm_comm_init")
        self._h = h
        w, r, d = C.c_int32(), C.c_int32(), C.c_int32()
        lib().spmm_comm_info(h, C.byref(w), C.byref(r), C.byref(d))
        self.world, self.rank, self.device = int(w.value), int(r.value), int(d.value)

    @property
    def handle(self):
        return self._h

    def close(self) -> None:
        if self._h:
            lib().spmm_comm_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


class RankPlan:
    """spmm_rank_plan_*: this rank's share of C = A @ B under the reference's nnz-balanced row split.

    A is the whole host CSR (the same on every rank); comm None is a world of one. run() is the
    end-to-end multiply from host buffers (collective), execute() the kernels alone on the
    device-resident operands the last run() left."""

    def __init__(self, comm: RankComm | None, A: HostCSR, N: int, stream=None):
        self._comm = comm
        self._A = A
        self.N = N
        v = A.view()
        h = C.c_void_p()
        check(lib().spmm_rank_plan_create(comm.handle if comm else None, C.byref(v), N, stream_ptr(stream),
                                          C.byref(h)), "spmm_rank_plan_create")
        self._h = h
        vals = [C.c_int32() for _ in range(7)]
        check(lib().spmm_rank_plan_info(h, *[C.byref(x) for x in vals]), "spmm_rank_plan_info")
        (self.row_begin, self.row_end, self.nnz, self.b_row_begin, self.b_row_end, self.algo,
         self.launches) = (int(x.value) for x in vals)
        dB, dC = C.c_void_p(), C.c_void_p()
        check(lib().spmm_rank_plan_buffers(h, C.byref(dB), C.byref(dC)), "spmm_rank_plan_buffers")
        self.d_B, self.d_C = int(dB.value or 0), int(dC.value or 0)

    @property
    def rows(self) -> int:
        return self.row_end - self.row_begin

    def run(self, A: HostCSR, B: np.ndarray, C_rows: np.ndarray, stream=None) -> None:
        v = A.view()
        check(lib().spmm_rank_run(self._h, C.byref(v), ptr(B), ptr(C_rows), stream_ptr(stream)), "spmm_rank_run")

    def submit(self, A: HostCSR, B: np.ndarray, C_rows: np.ndarray, stream=None) -> None:
        """run() without the wait; the arrays must stay alive and unchanged until wait()."""
        v = A.view()
        check(lib().spmm_rank_submit(self._h, C.byref(v), ptr(B), ptr(C_rows), stream_ptr(stream)),
              "spmm_rank_submit")

    def wait(self, stream=None) -> None:
        check(lib().spmm_rank_wait(self._h, stream_ptr(stream)), "spmm_rank_wait")

    def execute(self, stream=None) -> None:
        check(lib().spmm_rank_execute(self._h, stream_ptr(stream)), "spmm_rank_execute")

    def gather_b(self, stream=None) -> None:
        check(lib().spmm_rank_gather_b(self._h, stream_ptr(stream)), "spmm_rank_gather_b")

    def close(self) -> None:
        if self._h:
            lib().spmm_rank_plan_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:  # noqa: BLE001 - interpreter shutdown
            pass


# ------------------------------------------------------------------ rows grouped by an index
#
# Routing to experts and back, the experts' products, low-rank adapters (include/spmm_c.h says what each computes).
# Operands are torch tensors on the current CUDA device: rows may be strided, the elements of a row may not; index
# tensors (int32), weights (float32) and matrices are contiguous. Outputs are the caller's. A tensor of another
# type, shape or device raises ValueError, a refusal of the library SpmmError. `stream`: None is the legacy default
# stream, as everywhere here.

# The checks are a few attribute reads a tensor: at the sizes of single tokens they would otherwise cost more than the
# launch (a whole call is about 6 us of host time).

_torch = None  # the torch module, once a tensor has been seen
_DTYPES: dict = {}


def _device(t) -> int:
    """The current device, on which `t` and every other operand must be."""
    global _torch
    if _torch is None:
        import torch

        _DTYPES.update({torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16, torch.float32: DTYPE_F32})
        _torch = torch
    dev = t.get_device()
    if dev < 0 or dev != _torch._C._cuda_getDevice():  # current_device() without its check that CUDA is up
        raise ValueError(f"operands must be on the current CUDA device, got {t.device}")
    return dev


def _refuse(t, what: str, shape: tuple, dtype, dev: int):
    raise ValueError(f"{what}: want {shape} {dtype} on cuda:{dev}, got {tuple(t.shape)} {t.dtype}, strides {t.stride()}, on {t.device}")


def _rows(t, what: str, shape: tuple, dtype, dev: int) -> int:
    """Row stride of a (rows, columns) tensor whose rows are contiguous and do not overlap."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev:
        _refuse(t, what, shape, dtype, dev)
    ld, step = t.stride()
    if ld >= shape[1] and step == 1:
        return ld
    if (step != 1 and shape[1] > 1) or (ld < shape[1] and shape[0] > 1):
        _refuse(t, what + " (the elements of a row adjacent, rows apart)", shape, dtype, dev)
    return max(ld, shape[1])


def _flat(t, what: str, shape: tuple, dtype, dev: int) -> int:
    """Address of a contiguous tensor (0 for None)."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _refuse(t, what + " (contiguous)", shape, dtype, dev)
    return t.data_ptr()


def _value_dtype(t, what: str, f32: bool = False) -> int:
    dt = _DTYPES.get(t.dtype)
    if dt is None or (dt == DTYPE_F32 and not f32):
        raise ValueError(f"{what}: unsupported type {t.dtype}")
    return dt


def _workspace(ws, need: int, stream: int, dev: int):
    """(tensor that owns the workspace, address, bytes). Without one from the caller, memory of torch's allocator in the
    order of `stream`: reused by a later allocation only behind this call's kernels, also under graph capture."""
    if need == 0:
        return None, 0, 0
    if ws is None:
        cuda = _torch.cuda
        if stream == cuda.current_stream().cuda_stream:
            ws = _torch.empty(need, dtype=_torch.uint8, device="cuda")
        else:
            with cuda.stream(cuda.ExternalStream(stream) if stream else cuda.default_stream()):
                ws = _torch.empty(need, dtype=_torch.uint8, device="cuda")
    elif ws.get_device() != dev or not ws.is_contiguous():
        raise ValueError("ws: want a contiguous CUDA tensor on the current device")
    return ws, ws.data_ptr(), ws.numel() * ws.element_size()


@functools.lru_cache(maxsize=1024)
def route_workspace_size(tokens: int, topk: int, groups: int) -> int:
    n = C.c_size_t()
    check(lib().spmm_route_workspace_size(tokens, topk, groups, C.byref(n)), "spmm_route_workspace_size")
    return int(n.value)


def route_build(ids, groups: int, offsets, order, pos, ws=None, stream=None) -> None:
    """Sort the pairs of ids (tokens, topk) by group: offsets (groups + 1), order (tokens * topk, or None), pos (tokens, topk)."""
    dev = _device(ids)
    i32 = _torch.int32
    shape = tokens, topk = ids.shape
    sp = stream_ptr(stream)
    _ws, wp, wn = _workspace(ws, route_workspace_size(tokens, topk, groups), sp, dev)
    check(lib().spmm_route_build(_flat(ids, "ids", shape, i32, dev), tokens, topk, groups,
                                 _flat(offsets, "offsets", (groups + 1,), i32, dev),
                                 _flat(order, "order", (tokens * topk,), i32, dev), _flat(pos, "pos", shape, i32, dev), wp, wn, sp),
          "spmm_route_build")


_pack_route = struct.Struct("@iiiP").pack  # the bytes of a RouteView, in a third of its constructor's time
_pack_lora = struct.Struct("@iiiiiPPP").pack


def _route_view(pos, tokens: int, topk: int, rows: int, dev: int) -> bytes:
    return _pack_route(tokens, topk, rows, _flat(pos, "pos", (tokens, topk), _torch.int32, dev))


def route_gather(pos, x, xs, stream=None) -> None:
    """xs[pos[t, j]] = x[t] (rows of xs without a pair stay as they are)."""
    dev = _device(pos)
    tokens, topk = pos.shape
    shape = rows, H = xs.shape
    v = _route_view(pos, tokens, topk, rows, dev)
    check(lib().spmm_route_gather(v, x.data_ptr(), _rows(x, "x", (tokens, H), x.dtype, dev), xs.data_ptr(),
                                  _rows(xs, "xs", shape, x.dtype, dev), H, _value_dtype(x, "x", True), stream_ptr(stream)),
          "spmm_route_gather")


def route_combine(pos, ys, y, w=None, stream=None) -> None:
    """y[t] = sum_j w[t, j] ys[pos[t, j]] (w None: all 1, the gradient of route_gather)."""
    dev = _device(pos)
    tokens, topk = pos.shape
    shape = rows, H = ys.shape
    v = _route_view(pos, tokens, topk, rows, dev)
    check(lib().spmm_route_combine(v, ys.data_ptr(), _rows(ys, "ys", shape, ys.dtype, dev),
                                   _flat(w, "w", pos.shape, _torch.float32, dev), y.data_ptr(),
                                   _rows(y, "y", (tokens, H), ys.dtype, dev), H, _value_dtype(ys, "ys", True), stream_ptr(stream)),
          "spmm_route_combine")


def route_combine_grad(pos, dy, ys=None, w=None, dys=None, dw=None, stream=None) -> None:
    """Gradients of route_combine: dys[pos[t, j]] = w[t, j] dy[t] and dw[t, j] = <dy[t], ys[pos[t, j]]>; either may be left out
    (None; ys is needed for dw only)."""
    dev = _device(pos)
    if dys is None and dw is None:
        raise ValueError("route_combine_grad: neither dys nor dw is wanted")
    if dw is not None and ys is None:
        raise ValueError("route_combine_grad: dw needs ys")
    H = dy.shape[1]
    ys = ys if dw is not None else None
    shape = ((dys if dys is not None else ys).shape[0], H)
    tokens, topk = pos.shape
    v = _route_view(pos, tokens, topk, shape[0], dev)
    f32 = _torch.float32
    check(lib().spmm_route_combine_grad(
        v, dy.data_ptr(), _rows(dy, "dy", (tokens, H), dy.dtype, dev), ptr(ys),
        _rows(ys, "ys", shape, dy.dtype, dev) if ys is not None else 0, _flat(w, "w", pos.shape, f32, dev), ptr(dys),
        _rows(dys, "dys", shape, dy.dtype, dev) if dys is not None else 0, _flat(dw, "dw", pos.shape, f32, dev), H,
        _value_dtype(dy, "dy", True), stream_ptr(stream)), "spmm_route_combine_grad")


def grouped_mm(offsets, x, w, y, stream=None) -> None:
    """y[p] = w[g] x[p] for offsets[g] <= p < offsets[g + 1]; x (rows, K), w (groups, N, K), y (rows, N) of x's type or float32."""
    dev = _device(offsets)
    groups, N, K = w.shape
    rows = x.shape[0]
    check(lib().spmm_grouped_mm(_flat(offsets, "offsets", (groups + 1,), _torch.int32, dev), groups, rows, x.data_ptr(),
                                _rows(x, "x", (rows, K), x.dtype, dev), _flat(w, "w", w.shape, x.dtype, dev), y.data_ptr(),
                                _rows(y, "y", (rows, N), y.dtype, dev), N, K, _value_dtype(x, "x"), _value_dtype(y, "y", True),
                                stream_ptr(stream)), "spmm_grouped_mm")


def grouped_mm_dx(offsets, dy, w, dx, stream=None) -> None:
    """dx[p] = w[g]^T dy[p]; dy (rows, N), w (groups, N, K), dx (rows, K) of dy's type or float32."""
    dev = _device(offsets)
    groups, N, K = w.shape
    rows = dy.shape[0]
    check(lib().spmm_grouped_mm_dx(_flat(offsets, "offsets", (groups + 1,), _torch.int32, dev), groups, rows, dy.data_ptr(),
                                   _rows(dy, "dy", (rows, N), dy.dtype, dev), _flat(w, "w", w.shape, dy.dtype, dev), dx.data_ptr(),
                                   _rows(dx, "dx", (rows, K), dx.dtype, dev), N, K, _value_dtype(dy, "dy"),
                                   _value_dtype(dx, "dx", True), stream_ptr(stream)), "spmm_grouped_mm_dx")


def grouped_mm_dw(offsets, dy, x, dw, stream=None) -> None:
    """dw[g] = sum over the group's rows of dy[p] x[p]^T; dw (groups, N, K) of x's type or float32."""
    dev = _device(offsets)
    groups, N, K = dw.shape
    rows = x.shape[0]
    check(lib().spmm_grouped_mm_dw(_flat(offsets, "offsets", (groups + 1,), _torch.int32, dev), groups, rows, dy.data_ptr(),
                                   _rows(dy, "dy", (rows, N), x.dtype, dev), x.data_ptr(), _rows(x, "x", (rows, K), x.dtype, dev),
                                   _flat(dw, "dw", dw.shape, dw.dtype, dev), N, K, _value_dtype(x, "x"), _value_dtype(dw, "dw", True),
                                   stream_ptr(stream)), "spmm_grouped_mm_dw")


@functools.lru_cache(maxsize=1024)
def _lora_workspace(adapters: int, rank: int, N: int, K: int, dtype: int, requests: int, rows: int) -> int:
    v = LoraView(adapters, rank, N, K, dtype, 0, 0, 0)
    n = C.c_size_t()
    check(lib().spmm_lora_workspace_size(C.byref(v), requests, rows, C.byref(n)), "spmm_lora_workspace_size")
    return int(n.value)


def lora_workspace_size(a, b, requests: int, rows: int) -> int:
    _device(a)
    return _lora_workspace(a.shape[0], a.shape[1], b.shape[1], a.shape[2], _value_dtype(a, "a"), requests, rows)


def lora(offsets, adapter, x, a, b, out, base=None, scale=None, ws=None, stream=None) -> None:
    """out[p] = base[p] + scale * b (a x[p]) with the matrices of adapter[r], offsets[r] <= p < offsets[r + 1] (offsets None: every
    row a request of its own); x (rows, K), a (adapters, rank, K), b (adapters, N, rank), base and out (rows, N)."""
    dev = _device(adapter)
    shape = adapters, rank, K = a.shape
    N, rows, requests, dt = b.shape[1], x.shape[0], adapter.shape[0], _value_dtype(a, "a")
    v = _pack_lora(adapters, rank, N, K, dt, _flat(a, "a", shape, a.dtype, dev), _flat(b, "b", (adapters, N, rank), a.dtype, dev),
                   _flat(scale, "scale", (adapters,), _torch.float32, dev))
    sp, wide = stream_ptr(stream), (rows, N)
    _ws, wp, wn = _workspace(ws, _lora_workspace(adapters, rank, N, K, dt, requests, rows), sp, dev)
    check(lib().spmm_lora(v, _flat(offsets, "offsets", (requests + 1,), _torch.int32, dev),
                          _flat(adapter, "adapter", (requests,), _torch.int32, dev), requests, rows, x.data_ptr(),
                          _rows(x, "x", (rows, K), a.dtype, dev), ptr(base), _rows(base, "base", wide, a.dtype, dev) if base is not None else 0,
                          out.data_ptr(), _rows(out, "out", wide, a.dtype, dev), wp, wn, sp), "spmm_lora")
