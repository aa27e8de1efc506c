"""Python binding of the gfx950 VCSR SpMM library (lib/libvcsr_spmm.so).

A thin ctypes layer over the C ABI of include/vcsr_spmm.h, with the
reference's function names (MuuSeoTia/VCSR-SPMM) so callers and tests read
like the reference's host code:

    read_matrix_market_coo(path)          include/mmio.hpp:22
    coo_to_csr(coo)                       include/csr.hpp:16
    csr_to_vcsr_spmm(csr, segw, bundle)   include/vcsr.hpp:25    (layout H)
    csr_to_vcsr_seg(csr, segw, bundle)    src/vcsr_seg.cu:24     (layout S)
    csr_to_vcsr_opt(csr, segw, bundle)    src/vcsr_opt.cu:23     (layout S)
    csr_to_vcsr_tc(csr, bundle)           src/vcsr_tc.cu:26      (layout TC)
    run_csr_spmm_gpu(...)                 src/kernels.cu:107
    run_vcsr_spmm_gpu(fmt, dB, O, tileK, dC, stream)   src/kernels.cu:120
    run_vcsr_tc_spmm_gpu(fmt, dB, O, dC, stream)       src/vcsr_tc.cu:197

Errors: the reference throws std::runtime_error from the builders and exits
on CUDA errors; here every failure raises VcsrError carrying the library
status code and message.  GPU calls need a GPU: there is no CPU fallback,
and calling one without a GPU raises VcsrError (status VCSR_EDEVICE).
Device memory and streams are the library's own (DeviceArray, Stream); no
second GPU runtime is loaded into the process.
"""
from __future__ import annotations

import ctypes as C
import functools
import os
import struct
import threading

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "lib", "libvcsr_spmm.so")
CLI_PATH = os.path.join(_HERE, "bin", "spmm_vcsr")

VCSR_OK, VCSR_EINVAL, VCSR_EIO, VCSR_ENOMEM, VCSR_EDEVICE, VCSR_ERANGE, VCSR_ESTATE = range(7)
LAYOUT_H, LAYOUT_S, LAYOUT_TC = 0, 1, 2
KERNEL_AUTO, KERNEL_SEGMENT, KERNEL_MFMA, KERNEL_ROW, KERNEL_TILE = 0, 1, 2, 3, 4
# Value types of the dense operators as buffers carry them: float32, bf16 as
# 16-bit patterns, e4m3 as 8-bit patterns (VCSR_F32, VCSR_BF16, VCSR_FP8).
F32, BF16, FP8 = np.dtype(np.float32), np.dtype(np.uint16), np.dtype(np.uint8)
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}

# Every symbol include/vcsr_spmm.h declares (checked by the CPU test suite).
EXPORTS = (
    "vcsr_last_error vcsr_version vcsr_mtx_read vcsr_coo_create vcsr_coo_view_get "
    "vcsr_coo_free vcsr_gen_coo vcsr_gen_dense vcsr_coo_to_csr vcsr_csr_create "
    "vcsr_csr_view_get vcsr_csr_free vcsr_build vcsr_fmt_arrays vcsr_fmt_save vcsr_fmt_load "
    "vcsr_fmt_upload "
    "vcsr_fmt_set_tile_rows vcsr_fmt_set_tile_windows vcsr_fmt_tile_info vcsr_fmt_free spmm_csr_naive spmm_csr_wave spmm_vcsr "
    "spmm_vcsr_ex spmm_vcsr_noalloc spmm_vcsr_mfma vcsr_mfma_work vcsr_launch_info_get vcsr_tile_mfma_work spmm_csr_cpu "
    "vcsr_vendor_plan_create vcsr_vendor_spmm vcsr_vendor_plan_free spmm_csr_vendor "
    "vcsr_device_count vcsr_device_current vcsr_device_name vcsr_dev_malloc vcsr_dev_free "
    "vcsr_memcpy_h2d vcsr_memcpy_d2h vcsr_memcpy_d2d vcsr_memset_d vcsr_stream_create vcsr_stream_destroy "
    "vcsr_stream_sync vcsr_device_sync vcsr_event_create vcsr_event_destroy "
    "vcsr_event_record vcsr_event_elapsed "
    "vcsr_rmsnorm vcsr_rmsnorm_grad_workspace vcsr_rmsnorm_grad "
    "vcsr_layernorm vcsr_layernorm_grad_workspace vcsr_layernorm_grad "
    "vcsr_embed vcsr_embed_grad_workspace vcsr_embed_grad vcsr_linear_workspace vcsr_linear "
    "vcsr_linear_grad_workspace vcsr_linear_grad vcsr_gated_workspace vcsr_gated "
    "vcsr_gated_grad_workspace vcsr_gated_grad vcsr_adamw_create vcsr_adamw_step vcsr_adamw_free"
).split()


class VcsrError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"[{code}] {msg}")
        self.code = code


class _CooView(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("nnz", C.c_int64),
                ("rows", C.POINTER(C.c_int32)), ("cols", C.POINTER(C.c_int32)),
                ("vals", C.POINTER(C.c_float))]


class _CsrView(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("nnz", C.c_int32),
                ("row_ptr", C.POINTER(C.c_int32)), ("col", C.POINTER(C.c_int32)),
                ("val", C.POINTER(C.c_float))]


class _LaunchInfo(C.Structure):
    _fields_ = [("kernel", C.c_int32), ("tile_rows", C.c_int32), ("tiles", C.c_int64),
                ("entries", C.c_int64), ("matrix_cores", C.c_int32), ("vec", C.c_int32),
                ("column_slices", C.c_int32), ("slice_cols", C.c_int32),
                ("reduce_launches", C.c_int32), ("split_rows", C.c_int32),
                ("scratch_floats", C.c_int64)]


class _Arrays(C.Structure):
    _fields_ = [("M", C.c_int32), ("N", C.c_int32), ("segw", C.c_int32),
                ("bundle", C.c_int32), ("layout", C.c_int32), ("num_groups", C.c_int32),
                ("num_segments", C.c_int32), ("num_slots", C.c_int64),
                ("group_ptr", C.POINTER(C.c_int32)), ("group_depth", C.POINTER(C.c_int32)),
                ("group_seg_base", C.POINTER(C.c_int32)), ("group_rows", C.POINTER(C.c_int32)),
                ("lcol", C.POINTER(C.c_int32)), ("val", C.POINTER(C.c_float)),
                ("segment_group_start", C.POINTER(C.c_int32))]


class _RmsnormArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("C", C.c_int32), ("x_type", C.c_int32), ("y_type", C.c_int32),
                ("eps", C.c_float), ("x", C.c_void_p), ("ldx", C.c_int64),
                ("residual", C.c_void_p), ("ldr", C.c_int64), ("weight", C.c_void_p),
                ("sum", C.c_void_p), ("ldsum", C.c_int64), ("y", C.c_void_p), ("ldy", C.c_int64),
                ("y_scale", C.c_void_p), ("rstd", C.c_void_p)]


class _RmsnormGradArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("C", C.c_int32), ("x_type", C.c_int32), ("y_type", C.c_int32),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("s", C.c_void_p), ("lds", C.c_int64),
                ("weight", C.c_void_p), ("rstd", C.c_void_p), ("dsum", C.c_void_p),
                ("lddsum", C.c_int64), ("dx", C.c_void_p), ("lddx", C.c_int64),
                ("dweight", C.c_void_p), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


class _LayernormArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("C", C.c_int32), ("x_type", C.c_int32), ("y_type", C.c_int32),
                ("eps", C.c_float), ("x", C.c_void_p), ("ldx", C.c_int64),
                ("residual", C.c_void_p), ("ldr", C.c_int64), ("weight", C.c_void_p),
                ("bias", C.c_void_p), ("sum", C.c_void_p), ("ldsum", C.c_int64),
                ("y", C.c_void_p), ("ldy", C.c_int64), ("y_scale", C.c_void_p),
                ("mean", C.c_void_p), ("rstd", C.c_void_p)]


class _LayernormGradArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("C", C.c_int32), ("x_type", C.c_int32), ("y_type", C.c_int32),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("s", C.c_void_p), ("lds", C.c_int64),
                ("weight", C.c_void_p), ("mean", C.c_void_p), ("rstd", C.c_void_p),
                ("dsum", C.c_void_p), ("lddsum", C.c_int64), ("dx", C.c_void_p),
                ("lddx", C.c_int64), ("dweight", C.c_void_p), ("dbias", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class _EmbedArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("V", C.c_int32), ("C", C.c_int32), ("table_type", C.c_int32),
                ("y_type", C.c_int32), ("scale", C.c_float), ("table", C.c_void_p),
                ("ldt", C.c_int64), ("table_scale", C.c_void_p), ("ids", C.c_void_p),
                ("y", C.c_void_p), ("ldy", C.c_int64)]


class _EmbedGradArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("V", C.c_int32), ("C", C.c_int32), ("table_type", C.c_int32),
                ("y_type", C.c_int32), ("accumulate", C.c_int32), ("scale", C.c_float),
                ("dy", C.c_void_p), ("lddy", C.c_int64), ("ids", C.c_void_p),
                ("dtable", C.c_void_p), ("lddt", C.c_int64), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


class _LinearArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("N", C.c_int32), ("K", C.c_int32), ("x_type", C.c_int32),
                ("y_type", C.c_int32), ("act", C.c_int32), ("x", C.c_void_p), ("ldx", C.c_int64),
                ("w", C.c_void_p), ("ldw", C.c_int64), ("x_scale", C.c_void_p),
                ("w_scale", C.c_void_p), ("bias", C.c_void_p), ("residual", C.c_void_p),
                ("ldr", C.c_int64), ("z", C.c_void_p), ("ldz", C.c_int64), ("y", C.c_void_p),
                ("ldy", C.c_int64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class _LinearGradArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("N", C.c_int32), ("K", C.c_int32), ("x_type", C.c_int32),
                ("y_type", C.c_int32), ("act", C.c_int32), ("dy", C.c_void_p),
                ("lddy", C.c_int64), ("z", C.c_void_p), ("ldz", C.c_int64), ("x", C.c_void_p),
                ("ldx", C.c_int64), ("w", C.c_void_p), ("ldw", C.c_int64), ("dx", C.c_void_p),
                ("lddx", C.c_int64), ("dw", C.c_void_p), ("lddw", C.c_int64),
                ("dbias", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


class _GatedArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("N", C.c_int32), ("K", C.c_int32), ("x_type", C.c_int32),
                ("y_type", C.c_int32), ("act", C.c_int32), ("x", C.c_void_p), ("ldx", C.c_int64),
                ("w_gate", C.c_void_p), ("ldwg", C.c_int64), ("w_up", C.c_void_p),
                ("ldwu", C.c_int64), ("x_scale", C.c_void_p), ("gate_scale", C.c_void_p),
                ("up_scale", C.c_void_p), ("gate_bias", C.c_void_p), ("up_bias", C.c_void_p),
                ("z_gate", C.c_void_p), ("z_up", C.c_void_p), ("ldz", C.c_int64),
                ("y", C.c_void_p), ("ldy", C.c_int64), ("workspace", C.c_void_p),
                ("workspace_bytes", C.c_size_t)]


class _GatedGradArgs(C.Structure):
    _fields_ = [("M", C.c_int64), ("N", C.c_int32), ("K", C.c_int32), ("x_type", C.c_int32),
                ("y_type", C.c_int32), ("act", C.c_int32), ("dy", C.c_void_p),
                ("lddy", C.c_int64), ("z_gate", C.c_void_p), ("z_up", C.c_void_p),
                ("ldz", C.c_int64), ("x", C.c_void_p), ("ldx", C.c_int64),
                ("w_gate", C.c_void_p), ("ldwg", C.c_int64), ("w_up", C.c_void_p),
                ("ldwu", C.c_int64), ("dx", C.c_void_p), ("lddx", C.c_int64),
                ("dw_gate", C.c_void_p), ("lddwg", C.c_int64), ("dw_up", C.c_void_p),
                ("lddwu", C.c_int64), ("dgate_bias", C.c_void_p), ("dup_bias", C.c_void_p),
                ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)]


def _packer(fields, size):
    """struct.Struct of a ctypes structure's fields: packing costs a third of
    filling the structure, and a small call is bound by the host."""
    codes = {C.c_int64: "q", C.c_int32: "i", C.c_float: "f", C.c_void_p: "P", C.c_size_t: "N"}
    st = struct.Struct("@" + "".join(codes[t] for _, t in fields))
    assert st.size == size
    return st.pack


# The workspace's pointer and size end the structures that have them, and are packed
# by themselves.
_pack_rmsnorm = _packer(_RmsnormArgs._fields_, C.sizeof(_RmsnormArgs))
_pack_space = _packer(_LinearArgs._fields_[-2:], 16)
_pack_layernorm = _packer(_LayernormArgs._fields_, C.sizeof(_LayernormArgs))
_pack_embed = _packer(_EmbedArgs._fields_, C.sizeof(_EmbedArgs))
(_pack_rmsnorm_grad, _pack_layernorm_grad, _pack_embed_grad, _pack_linear, _pack_linear_grad,
 _pack_gated, _pack_gated_grad) = (
    _packer(args._fields_[:-2], C.sizeof(args) - 16)
    for args in (_RmsnormGradArgs, _LayernormGradArgs, _EmbedGradArgs, _LinearArgs,
                 _LinearGradArgs, _GatedArgs, _GatedGradArgs))


class _AdamwTensor(C.Structure):
    _fields_ = [("n", C.c_int64), ("grad_type", C.c_int32), ("state_type", C.c_int32),
                ("param", C.c_void_p), ("grad", C.c_void_p), ("m", C.c_void_p),
                ("v", C.c_void_p), ("m_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("copy", C.c_void_p), ("weight_decay", C.c_double)]


class _AdamwHyper(C.Structure):
    _fields_ = [("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double),
                ("eps", C.c_double), ("grad_scale", C.c_double), ("step", C.c_int64)]


_lib = None


def load_library(path: str = LIB_PATH) -> C.CDLL:
    """Loads lib/libvcsr_spmm.so; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise VcsrError(VCSR_EDEVICE, f"{path} not built (run __graft_entry__.build())")
    lib = C.CDLL(path)
    P, I32, I64, U64, F = C.c_void_p, C.c_int32, C.c_int64, C.c_uint64, C.c_float
    pI, pF, pP = C.POINTER(C.c_int32), C.POINTER(C.c_float), C.POINTER(C.c_void_p)
    pS = C.POINTER(C.c_size_t)
    sig = {
        "vcsr_last_error": (C.c_char_p, []),
        "vcsr_version": (C.c_char_p, []),
        "vcsr_mtx_read": (C.c_int, [C.c_char_p, I32, pP]),
        "vcsr_coo_create": (C.c_int, [I32, I32, I64, P, P, P, pP]),
        "vcsr_coo_view_get": (C.c_int, [P, C.POINTER(_CooView)]),
        "vcsr_coo_free": (None, [P]),
        "vcsr_gen_coo": (C.c_int, [I32, U64, pP]),
        "vcsr_gen_dense": (C.c_int, [U64, I32, I64, I32, P]),
        "vcsr_coo_to_csr": (C.c_int, [P, pP]),
        "vcsr_csr_create": (C.c_int, [I32, I32, P, P, P, pP]),
        "vcsr_csr_view_get": (C.c_int, [P, C.POINTER(_CsrView)]),
        "vcsr_csr_free": (None, [P]),
        "vcsr_build": (C.c_int, [P, I32, I32, I32, I32, pP]),
        "vcsr_fmt_arrays": (C.c_int, [P, C.POINTER(_Arrays)]),
        "vcsr_fmt_upload": (C.c_int, [P, P]),
        "vcsr_fmt_save": (C.c_int, [P, C.c_char_p]),
        "vcsr_fmt_load": (C.c_int, [C.c_char_p, pP]),
        "vcsr_fmt_set_tile_rows": (C.c_int, [P, I32]),
        "vcsr_fmt_set_tile_windows": (C.c_int, [P, I32]),
        "vcsr_fmt_tile_info": (C.c_int, [P, pI, C.POINTER(I64), C.POINTER(I64)]),
        "vcsr_fmt_free": (None, [P]),
        "spmm_csr_naive": (C.c_int, [I32, P, P, P, P, I32, P, P, pF]),
        "spmm_csr_wave": (C.c_int, [I32, I32, P, P, P, P, I32, P, P, pF]),
        "spmm_vcsr": (C.c_int, [P, P, I32, I32, P, P, pF]),
        "spmm_vcsr_ex": (C.c_int, [P, P, I32, I32, P, P, pF, I32, I32]),
        "spmm_vcsr_noalloc": (C.c_int, [P, P, I32, P, P, I32]),
        "spmm_vcsr_mfma": (C.c_int, [P, P, I32, P, P, pF]),
        "vcsr_mfma_work": (C.c_int, [P, I32, I32, C.POINTER(I64), pI]),
        "vcsr_launch_info_get": (C.c_int, [P, I32, I32, C.POINTER(_LaunchInfo)]),
        "vcsr_tile_mfma_work": (C.c_int, [P, I32, C.POINTER(I64), pI]),
        "spmm_csr_cpu": (C.c_int, [I32, P, P, P, P, I32, P, I32]),
        "vcsr_vendor_plan_create": (C.c_int, [I32, I32, I32, P, P, P, P, I32, P, P,
                                              C.POINTER(P)]),
        "vcsr_vendor_spmm": (C.c_int, [P, P, pF]),
        "vcsr_vendor_plan_free": (None, [P]),
        "spmm_csr_vendor": (C.c_int, [I32, I32, I32, P, P, P, P, I32, P, P, pF]),
        "vcsr_device_count": (C.c_int, [pI]),
        "vcsr_device_current": (C.c_int, [pI]),
        "vcsr_device_name": (C.c_int, [C.c_char_p, I32]),
        "vcsr_dev_malloc": (C.c_int, [pP, C.c_size_t]),
        "vcsr_dev_free": (C.c_int, [P]),
        "vcsr_memcpy_h2d": (C.c_int, [P, P, C.c_size_t, P]),
        "vcsr_memcpy_d2h": (C.c_int, [P, P, C.c_size_t, P]),
        "vcsr_memcpy_d2d": (C.c_int, [P, P, C.c_size_t, P]),
        "vcsr_memset_d": (C.c_int, [P, I32, C.c_size_t, P]),
        "vcsr_stream_create": (C.c_int, [pP]),
        "vcsr_stream_destroy": (C.c_int, [P]),
        "vcsr_stream_sync": (C.c_int, [P]),
        "vcsr_device_sync": (C.c_int, []),
        "vcsr_event_create": (C.c_int, [pP]),
        "vcsr_event_destroy": (C.c_int, [P]),
        "vcsr_event_record": (C.c_int, [P, P]),
        "vcsr_event_elapsed": (C.c_int, [P, P, pF]),
        "vcsr_rmsnorm": (C.c_int, [P, P, pF]),
        "vcsr_rmsnorm_grad_workspace": (C.c_int, [P, pS]),
        "vcsr_rmsnorm_grad": (C.c_int, [P, P, pF]),
        "vcsr_layernorm": (C.c_int, [P, P, pF]),
        "vcsr_layernorm_grad_workspace": (C.c_int, [P, pS]),
        "vcsr_layernorm_grad": (C.c_int, [P, P, pF]),
        "vcsr_embed": (C.c_int, [P, P, pF]),
        "vcsr_embed_grad_workspace": (C.c_int, [P, pS]),
        "vcsr_embed_grad": (C.c_int, [P, P, pF]),
        "vcsr_linear_workspace": (C.c_int, [P, pS]),
        "vcsr_linear": (C.c_int, [P, P, pF]),
        "vcsr_linear_grad_workspace": (C.c_int, [P, pS]),
        "vcsr_linear_grad": (C.c_int, [P, P, pF]),
        "vcsr_gated_workspace": (C.c_int, [P, pS]),
        "vcsr_gated": (C.c_int, [P, P, pF]),
        "vcsr_gated_grad_workspace": (C.c_int, [P, pS]),
        "vcsr_gated_grad": (C.c_int, [P, P, pF]),
        "vcsr_adamw_create": (C.c_int, [C.POINTER(_AdamwTensor), I32, P, pP]),
        "vcsr_adamw_step": (C.c_int, [P, C.POINTER(_AdamwHyper), P, pF]),
        "vcsr_adamw_free": (None, [P]),
    }
    for name, (res, args) in sig.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


def _check(rc: int) -> None:
    if rc != VCSR_OK:
        raise VcsrError(rc, load_library().vcsr_last_error().decode())


def _ptr(a: np.ndarray) -> C.c_void_p:
    return C.c_void_p(a.ctypes.data) if a.size else C.c_void_p(0)


def _copy(ptr, n: int, dtype) -> np.ndarray:
    if n == 0:
        return np.zeros(0, dtype=dtype)
    return np.ctypeslib.as_array(ptr, shape=(n,)).astype(dtype, copy=True)


# ----------------------------------------------------------------------- COO
class Coo:
    """Owned COO matrix (reference `struct COO`, include/mmio.hpp:15-19)."""

    def __init__(self, handle: C.c_void_p):
        self._h = handle
        v = _CooView()
        _check(load_library().vcsr_coo_view_get(self._h, C.byref(v)))
        self.M, self.N, self.nnz = v.M, v.N, v.nnz
        self.rows = _copy(v.rows, v.nnz, np.int32)
        self.cols = _copy(v.cols, v.nnz, np.int32)
        self.vals = _copy(v.vals, v.nnz, np.float32)

    def __del__(self):
        if getattr(self, "_h", None) and _lib is not None:
            _lib.vcsr_coo_free(self._h)
            self._h = None

    @staticmethod
    def from_arrays(M, N, rows, cols, vals) -> "Coo":
        rows = np.ascontiguousarray(rows, dtype=np.int32)
        cols = np.ascontiguousarray(cols, dtype=np.int32)
        vals = np.ascontiguousarray(vals, dtype=np.float32)
        h = C.c_void_p()
        _check(load_library().vcsr_coo_create(M, N, len(vals), _ptr(rows), _ptr(cols),
                                             _ptr(vals), C.byref(h)))
        return Coo(h)


def read_matrix_market_coo(path: str, expand_symmetric: bool = False) -> Coo:
    h = C.c_void_p()
    _check(load_library().vcsr_mtx_read(path.encode(), 1 if expand_symmetric else 0, C.byref(h)))
    return Coo(h)


def generate_coo(cfg: int, seed: int = 0) -> Coo:
    """Synthetic A of benchmark config cfg (1..5)."""
    h = C.c_void_p()
    _check(load_library().vcsr_gen_coo(cfg, seed, C.byref(h)))
    return Coo(h)


def gen_dense(seed: int, dist: int, rows: int, cols: int) -> np.ndarray:
    """Synthetic dense operand; dist 0 = U[-1,1), 1 = N(0,1)."""
    out = np.empty((rows, cols), dtype=np.float32)
    _check(load_library().vcsr_gen_dense(seed, dist, rows, cols, _ptr(out)))
    return out


# ----------------------------------------------------------------------- CSR
class Csr:
    """Owned CSR matrix (reference `struct CSR`, include/csr.hpp:8-13)."""

    def __init__(self, handle: C.c_void_p):
        self._h = handle
        v = _CsrView()
        _check(load_library().vcsr_csr_view_get(self._h, C.byref(v)))
        self.M, self.N, self.nnz = v.M, v.N, v.nnz
        self.row_ptr = _copy(v.row_ptr, v.M + 1, np.int32)
        self.col = _copy(v.col, v.nnz, np.int32)
        self.val = _copy(v.val, v.nnz, np.float32)

    def __del__(self):
        if getattr(self, "_h", None) and _lib is not None:
            _lib.vcsr_csr_free(self._h)
            self._h = None

    @staticmethod
    def from_arrays(M, N, row_ptr, col, val) -> "Csr":
        row_ptr = np.ascontiguousarray(row_ptr, dtype=np.int32)
        col = np.ascontiguousarray(col, dtype=np.int32)
        val = np.ascontiguousarray(val, dtype=np.float32)
        h = C.c_void_p()
        _check(load_library().vcsr_csr_create(M, N, _ptr(row_ptr), _ptr(col), _ptr(val),
                                             C.byref(h)))
        return Csr(h)


def coo_to_csr(coo: Coo) -> Csr:
    h = C.c_void_p()
    _check(load_library().vcsr_coo_to_csr(coo._h, C.byref(h)))
    return Csr(h)


# ---------------------------------------------------------------------- VCSR
class Vcsr:
    """Owned VCSR format; .arrays() returns copies of the packed arrays."""

    def __init__(self, handle: C.c_void_p):
        self._h = handle
        a = _Arrays()
        _check(load_library().vcsr_fmt_arrays(self._h, C.byref(a)))
        self.M, self.N, self.segw, self.bundle = a.M, a.N, a.segw, a.bundle
        self.layout, self.num_groups, self.num_segments = a.layout, a.num_groups, a.num_segments
        self.num_slots = a.num_slots

    def __del__(self):
        self.free()

    def free(self):
        if getattr(self, "_h", None) and _lib is not None:
            _lib.vcsr_fmt_free(self._h)
            self._h = None

    def arrays(self) -> dict:
        a = _Arrays()
        _check(load_library().vcsr_fmt_arrays(self._h, C.byref(a)))
        G, P, S, b = a.num_groups, a.num_slots, a.num_segments, a.bundle
        return {
            "group_ptr": _copy(a.group_ptr, G + 1, np.int32),
            "group_depth": _copy(a.group_depth, G, np.int32),
            "group_seg_base": _copy(a.group_seg_base, G, np.int32),
            "group_rows": _copy(a.group_rows, G * b, np.int32),
            "lcol": _copy(a.lcol, P, np.int32),
            "val": _copy(a.val, P, np.float32),
            "segment_group_start": _copy(a.segment_group_start, S + 1, np.int32),
        }

    def upload(self, stream: "Stream | None" = None) -> None:
        _check(load_library().vcsr_fmt_upload(self._h, _sp(stream)))

    def set_tile_rows(self, rows: int) -> None:
        """Tile height of the row-tile view (0 = automatic); before upload()."""
        _check(load_library().vcsr_fmt_set_tile_rows(self._h, rows))

    def set_tile_windows(self, fixed: bool) -> None:
        """Fixed row windows of the tile height instead of shared-column
        tiles (16 rows: FastSpMM's condensed tiles); before upload()."""
        _check(load_library().vcsr_fmt_set_tile_windows(self._h, 1 if fixed else 0))

    def launch_info(self, O: int, kernel: int = 0) -> dict:
        """What one SpMM of width O launches (vcsr_launch_info_get): kernel,
        row-tile view, column slices, reduce launches, scratch floats."""
        info = _LaunchInfo()
        _check(load_library().vcsr_launch_info_get(self._h, O, kernel, C.byref(info)))
        return {name: getattr(info, name) for name, _ in _LaunchInfo._fields_}

    def tile_info(self) -> tuple[int, int, int]:
        """(tile height, tiles, entries) of the uploaded row-tile view."""
        r, t, e = C.c_int32(), C.c_int64(), C.c_int64()
        _check(load_library().vcsr_fmt_tile_info(self._h, C.byref(r), C.byref(t), C.byref(e)))
        return r.value, t.value, e.value


def save_vcsr(fmt: "Vcsr", path: str) -> None:
    """Write the format (host arrays, tile-view settings) to a file."""
    _check(load_library().vcsr_fmt_save(fmt._h, os.fsencode(path)))


def load_vcsr(path: str) -> "Vcsr":
    """Read a format file written by save_vcsr (validated; not uploaded)."""
    h = C.c_void_p()
    _check(load_library().vcsr_fmt_load(os.fsencode(path), C.byref(h)))
    return Vcsr(h)


def build_vcsr(csr: Csr, segw: int, bundle: int, layout: int, nthreads: int = 0) -> Vcsr:
    h = C.c_void_p()
    _check(load_library().vcsr_build(csr._h, segw, bundle, layout, nthreads, C.byref(h)))
    return Vcsr(h)


def csr_to_vcsr_spmm(csr: Csr, segw: int = 4, bundle: int = 32) -> Vcsr:
    return build_vcsr(csr, segw, bundle, LAYOUT_H)


def csr_to_vcsr_seg(csr: Csr, segw: int, bundle: int) -> Vcsr:
    return build_vcsr(csr, segw, bundle, LAYOUT_S)


csr_to_vcsr_opt = csr_to_vcsr_seg


def csr_to_vcsr_tc(csr: Csr, bundle: int = 16) -> Vcsr:
    return build_vcsr(csr, 16, bundle, LAYOUT_TC)


def spmm_csr_cpu(csr: Csr, B: np.ndarray, nthreads: int = 0) -> np.ndarray:
    B = np.ascontiguousarray(B, dtype=np.float32)
    O = B.shape[1]
    out = np.empty((csr.M, O), dtype=np.float32)
    _check(load_library().spmm_csr_cpu(csr.M, _ptr(csr.row_ptr), _ptr(csr.col), _ptr(csr.val),
                                       _ptr(B), O, _ptr(out), nthreads))
    return out


# -------------------------------------------------------------------- device
def device_count() -> int:
    n = C.c_int32(0)
    _check(load_library().vcsr_device_count(C.byref(n)))
    return n.value


def current_device() -> int:
    d = C.c_int32(0)
    _check(load_library().vcsr_device_current(C.byref(d)))
    return d.value


def device_name() -> str:
    buf = C.create_string_buffer(128)
    _check(load_library().vcsr_device_name(buf, 128))
    return buf.value.decode()


class Stream:
    def __init__(self):
        self.h = C.c_void_p()
        _check(load_library().vcsr_stream_create(C.byref(self.h)))

    def sync(self):
        _check(load_library().vcsr_stream_sync(self.h))

    def __del__(self):
        if getattr(self, "h", None) and _lib is not None and self.h.value:
            # The next stream may get this one's handle, and its workspace with it.
            if _workspaces and any(key[1] == self.h.value for key in list(_workspaces)):
                _lib.vcsr_stream_sync(self.h)
            _lib.vcsr_stream_destroy(self.h)
            self.h = C.c_void_p()


def _sp(stream):
    return stream.h if stream is not None else C.c_void_p(0)


class Event:
    def __init__(self):
        self.h = C.c_void_p()
        _check(load_library().vcsr_event_create(C.byref(self.h)))

    def record(self, stream=None):
        _check(load_library().vcsr_event_record(self.h, _sp(stream)))

    def elapsed_ms(self, stop: "Event") -> float:
        ms = C.c_float(0)
        _check(load_library().vcsr_event_elapsed(self.h, stop.h, C.byref(ms)))
        return ms.value

    def __del__(self):
        if getattr(self, "h", None) and _lib is not None and self.h.value:
            _lib.vcsr_event_destroy(self.h)
            self.h = C.c_void_p()


class DeviceArray:
    """A device buffer owned by the library's HIP runtime."""

    def __init__(self, shape, dtype):
        self.shape = tuple(shape) if isinstance(shape, (tuple, list)) else (int(shape),)
        self.dtype = np.dtype(dtype)
        self.nbytes = int(np.prod(self.shape)) * self.dtype.itemsize
        self.ptr = C.c_void_p()
        _check(load_library().vcsr_dev_malloc(C.byref(self.ptr), self.nbytes))

    @staticmethod
    def from_numpy(a: np.ndarray, stream=None) -> "DeviceArray":
        a = np.ascontiguousarray(a)
        d = DeviceArray(a.shape, a.dtype)
        _check(load_library().vcsr_memcpy_h2d(d.ptr, _ptr(a), d.nbytes, _sp(stream)))
        return d

    def numpy(self, stream=None) -> np.ndarray:
        out = np.empty(self.shape, dtype=self.dtype)
        _check(load_library().vcsr_memcpy_d2h(_ptr(out), self.ptr, self.nbytes, _sp(stream)))
        return out

    def copy_from(self, other: "DeviceArray", stream=None) -> None:
        """Device-to-device copy of min(nbytes) bytes, enqueued on stream."""
        n = min(self.nbytes, other.nbytes)
        _check(load_library().vcsr_memcpy_d2d(self.ptr, other.ptr, n, _sp(stream)))

    def zero(self, stream=None) -> None:
        _check(load_library().vcsr_memset_d(self.ptr, 0, self.nbytes, _sp(stream)))

    def __del__(self):
        if getattr(self, "ptr", None) and _lib is not None and self.ptr.value:
            _lib.vcsr_dev_free(self.ptr)
            self.ptr = C.c_void_p()


def _need_buf(arr, dtype, count, what):
    """Raises VcsrError(VCSR_EINVAL) unless the device buffer `arr` holds at
    least `count` elements of `dtype`: the kernels index B and C by the
    shapes they are given, so a short or mistyped buffer would be read or
    written past its end on the device."""
    want = np.dtype(dtype)
    have = getattr(arr, "dtype", want)
    if np.dtype(have) != want:
        raise VcsrError(VCSR_EINVAL, f"{what}: dtype {np.dtype(have)}, expected {want}")
    nbytes = getattr(arr, "nbytes", None)
    if nbytes is None or int(nbytes) < int(count) * want.itemsize:
        raise VcsrError(VCSR_EINVAL, f"{what}: {nbytes} bytes, need {int(count) * want.itemsize}")


def _need_csr(M, d_rowptr, d_col, d_val, nnz=0):
    """CSR device buffers: row_ptr of M + 1 entries, col and val of equal
    length and at least `nnz` entries (the vendor library is told nnz and
    reads that many)."""
    if nnz < 0:
        raise VcsrError(VCSR_EINVAL, "negative nnz")
    _need_buf(d_rowptr, np.int32, M + 1, "row_ptr")
    _need_buf(d_col, np.int32, nnz, "col")
    _need_buf(d_val, np.float32, nnz, "val")
    if d_col.nbytes // 4 != d_val.nbytes // 4:
        raise VcsrError(VCSR_EINVAL, "col and val lengths differ")


def _need_bc(N, M, O, dB, dC):
    if O < 0:
        raise VcsrError(VCSR_EINVAL, "negative O")
    _need_buf(dB, np.float32, N * O, "B")
    _need_buf(dC, np.float32, M * O, "C")


def run_csr_spmm_gpu(M, d_rowptr, d_col, d_val, dB, O, dC, stream=None, timed=False):
    """C = A*B (overwrites C).  Returns kernel ms when timed (synchronous)."""
    _need_csr(M, d_rowptr, d_col, d_val)
    _need_bc(0, M, O, dB, dC)
    ms = C.c_float(0)
    _check(load_library().spmm_csr_naive(M, d_rowptr.ptr, d_col.ptr, d_val.ptr, dB.ptr, O,
                                         dC.ptr, _sp(stream), C.byref(ms) if timed else None))
    return ms.value if timed else None


class VendorPlan:
    """rocSPARSE SpMM (C = A*B) bound to device CSR arrays, B and C: the
    vendor baseline (the reference's run_cusparse_spmm, src/kernels.cu:169-235)
    with its set-up done once."""

    def __init__(self, M, N, nnz, d_rowptr, d_col, d_val, dB, O, dC, stream=None):
        _need_csr(M, d_rowptr, d_col, d_val, nnz)
        _need_bc(N, M, O, dB, dC)
        h = C.c_void_p()
        _check(load_library().vcsr_vendor_plan_create(M, N, nnz, d_rowptr.ptr, d_col.ptr,
                                                      d_val.ptr, dB.ptr, O, dC.ptr, _sp(stream),
                                                      C.byref(h)))
        self._h = h
        self._keep = (d_rowptr, d_col, d_val, dB, dC)

    def run(self, stream=None, timed=False):
        """C = A*B; the SpMM call's ms when timed (synchronous)."""
        ms = C.c_float(0)
        _check(load_library().vcsr_vendor_spmm(self._h, _sp(stream),
                                               C.byref(ms) if timed else None))
        return ms.value if timed else None

    def __del__(self):
        if getattr(self, "_h", None) and self._h.value:
            load_library().vcsr_vendor_plan_free(self._h)
            self._h = C.c_void_p()


def run_vendor_spmm_gpu(M, N, nnz, d_rowptr, d_col, d_val, dB, O, dC, stream=None, timed=False):
    """One-shot rocSPARSE C = A*B (set-up, SpMM, tear-down, like the
    reference's cuSPARSE wrapper); the SpMM call's ms when timed."""
    _need_csr(M, d_rowptr, d_col, d_val, nnz)
    _need_bc(N, M, O, dB, dC)
    ms = C.c_float(0)
    _check(load_library().spmm_csr_vendor(M, N, nnz, d_rowptr.ptr, d_col.ptr, d_val.ptr, dB.ptr,
                                          O, dC.ptr, _sp(stream), C.byref(ms) if timed else None))
    return ms.value if timed else None


def run_csr_wave_spmm_gpu(M, N, d_rowptr, d_col, d_val, dB, O, dC, stream=None, timed=False):
    """C = A*B with the wave-per-row CSR kernel (overwrites C); kernel ms
    when timed (synchronous)."""
    _need_csr(M, d_rowptr, d_col, d_val)
    _need_bc(N, M, O, dB, dC)
    ms = C.c_float(0)
    _check(load_library().spmm_csr_wave(M, N, d_rowptr.ptr, d_col.ptr, d_val.ptr, dB.ptr, O,
                                        dC.ptr, _sp(stream), C.byref(ms) if timed else None))
    return ms.value if timed else None


def run_vcsr_spmm_gpu(fmt: Vcsr, dB, O, tileK, dC, stream=None, timed=False):
    """C += A*B (spmm_vcsr: the default kernel, the reference's accumulate
    semantics, so zero C first)."""
    _need_bc(fmt.N, fmt.M, O, dB, dC)
    ms = C.c_float(0)
    _check(load_library().spmm_vcsr(fmt._h, dB.ptr, O, tileK, dC.ptr, _sp(stream),
                                    C.byref(ms) if timed else None))
    return ms.value if timed else None


def run_vcsr_tc_spmm_gpu(fmt: Vcsr, dB, O, dC, stream=None, timed=False):
    """C += A*B with the FP32-MFMA dense-tile kernel; zero C first."""
    _need_bc(fmt.N, fmt.M, O, dB, dC)
    ms = C.c_float(0)
    _check(load_library().spmm_vcsr_mfma(fmt._h, dB.ptr, O, dC.ptr, _sp(stream),
                                         C.byref(ms) if timed else None))
    return ms.value if timed else None


run_vcsr_mfma_spmm_gpu = run_vcsr_tc_spmm_gpu


def mfma_work(fmt: Vcsr, O: int, tileK: int = 0) -> tuple[int, int]:
    """(MFMA instructions, FLOPs per instruction) the FP32-MFMA kernel issues
    for one SpMM of width O (host only)."""
    ops, fpo = C.c_int64(), C.c_int32()
    _check(load_library().vcsr_mfma_work(fmt._h, O, tileK, C.byref(ops), C.byref(fpo)))
    return ops.value, fpo.value


def tile_mfma_work(fmt: Vcsr, O: int) -> tuple[int, int]:
    """(MFMA instructions, FLOPs per instruction) the tile-stationary kernel
    issues for one SpMM of width O on an uploaded format with 16-row tiles
    ((0, flops) for other tile heights)."""
    ops, fpo = C.c_int64(), C.c_int32()
    _check(load_library().vcsr_tile_mfma_work(fmt._h, O, C.byref(ops), C.byref(fpo)))
    return ops.value, fpo.value


def run_vcsr_spmm_gpu_ex(fmt: Vcsr, dB, O, tileK, dC, stream=None, timed=False,
                         kernel=KERNEL_AUTO, accumulate=True):
    """SpMM with an explicit kernel; accumulate=False computes C = A*B."""
    _need_bc(fmt.N, fmt.M, O, dB, dC)
    ms = C.c_float(0)
    _check(load_library().spmm_vcsr_ex(fmt._h, dB.ptr, O, tileK, dC.ptr, _sp(stream),
                                       C.byref(ms) if timed else None, kernel,
                                       1 if accumulate else 0))
    return ms.value if timed else None


def run_vcsr_spmm_gpu_noalloc(fmt: Vcsr, dB, O, dC, stream=None, accumulate=False):
    """The default (tile-stationary) kernel through spmm_vcsr_noalloc: no
    device allocation in the call; the partial rows of split tiles live in
    the library's fixed 16 MiB per-device scratch array (VCSR_ERANGE beyond
    it).  Enqueued only (not waited for); calls that overlap on one GPU race
    on that scratch."""
    _need_bc(fmt.N, fmt.M, O, dB, dC)
    _check(load_library().spmm_vcsr_noalloc(fmt._h, dB.ptr, O, dC.ptr, _sp(stream),
                                            1 if accumulate else 0))


# ----------------------------------------------------------- dense operators
class DeviceView:
    """A matrix or vector in device memory that another object owns (`owner`
    is kept alive): its address, shape, dtype (F32, BF16 or FP8) and, for a
    matrix, the elements from one row to the next."""

    def __init__(self, ptr, shape, dtype, ld=None, owner=None):
        self.ptr = C.c_void_p(int(getattr(ptr, "value", ptr) or 0))
        self.shape = tuple(shape) if isinstance(shape, (tuple, list)) else (int(shape),)
        self.dtype = np.dtype(dtype)
        self.ld = int(ld) if ld is not None else (self.shape[-1] if self.shape else 1)
        rows = int(np.prod(self.shape[:-1])) if len(self.shape) > 1 else 1
        elems = (rows - 1) * self.ld + self.shape[-1] if rows and self.shape else 0
        self.nbytes = elems * self.dtype.itemsize
        self.owner = owner


def to_bf16(a) -> np.ndarray:
    """float32 values as bf16 bit patterns (BF16), rounded to nearest even."""
    a = np.ascontiguousarray(a, np.float32)
    u = a.view(np.uint32)
    rounded = (u + 0x7FFF + ((u >> 16) & 1)) >> 16  # no carry past 32 bits but from a NaN
    return np.where(np.isnan(a), 0x7FC0, rounded).astype(BF16)


def from_bf16(u) -> np.ndarray:
    return (np.asarray(u, BF16).astype(np.uint32) << 16).view(np.float32)


def _e4m3_values():
    c = np.arange(128)
    e, m = c >> 3, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[127] = np.nan
    return np.concatenate([v, -v]).astype(np.float32)


_E4M3 = _e4m3_values()


def from_fp8(u) -> np.ndarray:
    """The values of e4m3 codes (FP8)."""
    return _E4M3[np.asarray(u, FP8)]


def quantize_fp8(a):
    """A matrix as e4m3 codes (FP8) and one float32 scale a row, as run_rmsnorm_gpu
    writes them: scale = max(max |row|, 1e-30) / 448, codes a / scale rounded to
    nearest even.  For weights that are laid out once; finite values only."""
    a = np.ascontiguousarray(a, np.float32)
    scale = np.maximum(np.abs(a).max(axis=1, initial=0), np.float32(1e-30)) / np.float32(448)
    x = np.minimum(np.abs(a / scale[:, None]), np.float32(448)).astype(np.float64)
    # The distance between neighbouring codes, from the value's exponent.
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(x, 2.0 ** -9))), -6) - 3)
    v = np.round(x / step) * step  # numpy rounds halves to even
    codes = np.searchsorted(_E4M3[:127], v).astype(FP8) | np.where(a < 0, 128, 0).astype(FP8)
    return codes, scale


_TYPE = {F32: 0, BF16: 1, FP8: 2}


def _type(arr, what):
    t = _TYPE.get(arr.dtype)
    if t is None:
        raise VcsrError(VCSR_EINVAL, f"{what}: dtype {arr.dtype}; float32, bf16 (uint16) or "
                                     "e4m3 (uint8) patterns are expected")
    return t


def _mat(arr, rows, cols, what, dtype=None):
    """(address, row stride) of a matrix argument after checking its shape,
    type and size; (0, 0) for None."""
    if arr is None:
        return 0, 0
    if arr.shape != (rows, cols):
        raise VcsrError(VCSR_EINVAL, f"{what}: shape {arr.shape}, expected {(rows, cols)}")
    have = arr.dtype
    if dtype is not None and have is not dtype and have != dtype:
        raise VcsrError(VCSR_EINVAL, f"{what}: dtype {have}, expected {dtype}")
    ld = getattr(arr, "ld", cols)
    if rows and arr.nbytes < ((rows - 1) * ld + cols) * have.itemsize:
        raise VcsrError(VCSR_EINVAL, f"{what}: {arr.nbytes} bytes are too few")
    return arr.ptr.value or 0, ld


def _vec(arr, n, what):
    if arr is None:
        return 0
    if (arr.dtype is not F32 and arr.dtype != F32) or arr.nbytes < 4 * n:
        raise VcsrError(VCSR_EINVAL, f"{what}: {arr.dtype}, {arr.nbytes} bytes; "
                                     f"{n} float32 values are expected")
    return arr.ptr.value or 0


def _ids(arr, what):
    """(address, count) of int32 indices, back to back."""
    if arr.dtype != np.int32 or len(arr.shape) != 1 or arr.nbytes < 4 * arr.shape[0]:
        raise VcsrError(VCSR_EINVAL, f"{what}: {arr.dtype} {arr.shape}, {arr.nbytes} bytes; a "
                                     "vector of int32 is expected")
    return arr.ptr.value or 0, arr.shape[0]


def _shape2(arr, what):
    if len(arr.shape) != 2:
        raise VcsrError(VCSR_EINVAL, f"{what}: shape {arr.shape}, a matrix is expected")
    return arr.shape


# (device, stream handle) -> DeviceArray; the buffers that these replaced, by device.
_workspaces, _outgrown = {}, {}
# Held from the choice of a workspace until the call that uses it has enqueued its
# kernels: between those of two host threads on one stream nothing else may write it.
_workspace_lock = threading.RLock()
_one_device = None  # whether the process sees a single device


def _device():
    global _one_device
    if _one_device is None:
        _one_device = device_count() <= 1
    return 0 if _one_device else current_device()


def workspace(nbytes, stream=None):
    """The binding's workspace of a stream on the current device, at least nbytes
    large.  Calls on one stream run one after the other, so they share it.  A call
    that needs more gets a larger one; the one before stays allocated, since work
    under way or a captured graph may use it, until release_workspaces().  A call
    that is captured into a graph takes the workspace that is there: make the same
    call once before the capture, and replay the graph on the stream it was captured
    on; for replays elsewhere, beside other calls, pass a DeviceArray of its own."""
    key = (_device(), stream.h.value if stream is not None else None)
    with _workspace_lock:
        have = _workspaces.get(key)
        if have is None or have.nbytes < nbytes:
            size = max(int(nbytes), 1 << 20)
            if have is None:
                new = DeviceArray((size,), np.uint8)
            else:
                try:  # twice as large, so that all that were outgrown take less than the last
                    new = DeviceArray((max(size, 2 * have.nbytes),), np.uint8)
                except VcsrError:
                    new = DeviceArray((size,), np.uint8)
                _outgrown.setdefault(key[0], []).append(have)
            have = _workspaces[key] = new
        return have


def release_workspaces():
    """Frees the current device's workspaces, those of all its streams, once the
    device is idle; no graph captured with them may be replayed any more."""
    device = _device()
    with _workspace_lock:
        mine = [key for key in _workspaces if key[0] == device]
        if mine:
            _check(load_library().vcsr_device_sync())
            for key in mine:
                del _workspaces[key]
            _outgrown.pop(device, None)


# Bytes of workspace by sizes and types alone (what the _workspace functions
# answer), so that a call asks the library once for each.
@functools.lru_cache(maxsize=4096)
def _linear_bytes(M, N, K, x_type, y_type, residual, z):
    need = C.c_size_t(0)
    args = _LinearArgs(M=M, N=N, K=K, x_type=x_type, y_type=y_type,
                       residual=16 if residual else None, z=16 if z else None)
    _check(load_library().vcsr_linear_workspace(C.byref(args), C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _linear_grad_bytes(M, N, K, x_type, y_type, act, z, dx, dw, dbias):
    need = C.c_size_t(0)
    some = C.c_void_p(16)
    args = _LinearGradArgs(M=M, N=N, K=K, x_type=x_type, y_type=y_type, act=act,
                           z=some if z else None, dx=some if dx else None,
                           dw=some if dw else None, dbias=some if dbias else None)
    _check(load_library().vcsr_linear_grad_workspace(C.byref(args), C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _rmsnorm_grad_bytes(M, N, x_type, y_type):
    need = C.c_size_t(0)
    args = _RmsnormGradArgs(M=M, C=N, x_type=x_type, y_type=y_type, dweight=16)
    _check(load_library().vcsr_rmsnorm_grad_workspace(C.byref(args), C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _layernorm_grad_bytes(M, N, x_type, y_type, dweight, dbias):
    need = C.c_size_t(0)
    args = _LayernormGradArgs(M=M, C=N, x_type=x_type, y_type=y_type,
                              dweight=16 if dweight else None, dbias=32 if dbias else None)
    _check(load_library().vcsr_layernorm_grad_workspace(C.byref(args), C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _embed_grad_bytes(M, V, N, table_type, y_type, accumulate):
    need = C.c_size_t(0)
    args = _EmbedGradArgs(M=M, V=V, C=N, table_type=table_type, y_type=y_type,
                          accumulate=accumulate)
    _check(load_library().vcsr_embed_grad_workspace(C.byref(args), C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _gated_bytes(M, N, K, x_type, y_type, z):
    need = C.c_size_t(0)
    args = _GatedArgs(M=M, N=N, K=K, x_type=x_type, y_type=y_type, z_gate=16 if z else None,
                      z_up=32 if z else None)
    _check(load_library().vcsr_gated_workspace(C.byref(args), C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _gated_grad_bytes(M, N, K, x_type, y_type, dx, dw, dgate_bias, dup_bias):
    need = C.c_size_t(0)
    args = _GatedGradArgs(M=M, N=N, K=K, x_type=x_type, y_type=y_type, dx=16 if dx else None,
                          dw_gate=32 if dw else None, dw_up=48 if dw else None,
                          dgate_bias=64 if dgate_bias else None,
                          dup_bias=80 if dup_bias else None)
    _check(load_library().vcsr_gated_grad_workspace(C.byref(args), C.byref(need)))
    return need.value


def _call(fn, args, stream, timed):
    if not timed:
        rc = fn(args, stream.h if stream is not None else None, None)
        if rc:
            _check(rc)
        return None
    ms = C.c_float(0)
    _check(fn(args, _sp(stream), C.byref(ms)))
    return ms.value


def _call_with_space(fn, args, need, given, stream, timed):
    """_call with `need` bytes of workspace, whose two fields end the structure:
    `given`, or the binding's own."""
    if not need:
        return _call(fn, args + _pack_space(0, 0), stream, timed)
    if given is not None:
        return _call(fn, args + _pack_space(given.ptr.value or 0, given.nbytes), stream, timed)
    with _workspace_lock:
        own = workspace(need, stream)
        return _call(fn, args + _pack_space(own.ptr.value, own.nbytes), stream, timed)


def run_rmsnorm_gpu(x, weight, y, residual=None, sum=None, y_scale=None, rstd=None, eps=1e-6,
                    stream=None, timed=False):
    """y = t / sqrt(mean(t^2) + eps) * weight for t = x + residual, row by row
    (vcsr_rmsnorm).  x, residual, sum: float32 or BF16; y: float32, BF16 or FP8
    with y_scale, one scale a row.  sum receives t, rstd each row's factor."""
    M, N = _shape2(x, "x")
    (xp, ldx), (rp, ldr) = _mat(x, M, N, "x"), _mat(residual, M, N, "residual", x.dtype)
    (sp, lds), (yp, ldy) = _mat(sum, M, N, "sum", x.dtype), _mat(y, M, N, "y")
    args = _pack_rmsnorm(M, N, _type(x, "x"), _type(y, "y"), eps, xp, ldx, rp, ldr,
                         _vec(weight, N, "weight"), sp, lds, yp, ldy,
                         _vec(y_scale, M, "y_scale"), _vec(rstd, M, "rstd"))
    return _call((_lib or load_library()).vcsr_rmsnorm, args, stream, timed)


def run_rmsnorm_grad_gpu(dy, s, weight, rstd, dx, dweight=None, dsum=None, workspace=None,
                         stream=None, timed=False):
    """Gradients of run_rmsnorm_gpu (vcsr_rmsnorm_grad): s is the saved sum (x
    without a residual), dsum what flows into it from elsewhere; dx is the
    gradient of x and of the residual."""
    M, N = _shape2(s, "s")
    (dp, lddy), (sp, lds) = _mat(dy, M, N, "dy"), _mat(s, M, N, "s")
    (up, ldu), (xp, ldx) = _mat(dsum, M, N, "dsum", s.dtype), _mat(dx, M, N, "dx", s.dtype)
    xt, yt = _type(s, "s"), _type(dy, "dy")
    need = _rmsnorm_grad_bytes(M, N, xt, yt) if dweight is not None else 0
    args = _pack_rmsnorm_grad(M, N, xt, yt, dp, lddy, sp, lds, _vec(weight, N, "weight"),
                              _vec(rstd, M, "rstd"), up, ldu, xp, ldx,
                              _vec(dweight, N, "dweight"))
    return _call_with_space((_lib or load_library()).vcsr_rmsnorm_grad, args, need, workspace,
                            stream, timed)


def run_layernorm_gpu(x, weight, y, bias=None, residual=None, sum=None, y_scale=None, mean=None,
                      rstd=None, eps=1e-5, stream=None, timed=False):
    """y = (t - mean(t)) / sqrt(var(t) + eps) * weight + bias for t = x + residual,
    row by row (vcsr_layernorm).  Types as run_rmsnorm_gpu's; sum receives t, mean and
    rstd each row's mean and factor."""
    M, N = _shape2(x, "x")
    (xp, ldx), (rp, ldr) = _mat(x, M, N, "x"), _mat(residual, M, N, "residual", x.dtype)
    (sp, lds), (yp, ldy) = _mat(sum, M, N, "sum", x.dtype), _mat(y, M, N, "y")
    args = _pack_layernorm(M, N, _type(x, "x"), _type(y, "y"), eps, xp, ldx, rp, ldr,
                           _vec(weight, N, "weight"), _vec(bias, N, "bias"), sp, lds, yp, ldy,
                           _vec(y_scale, M, "y_scale"), _vec(mean, M, "mean"),
                           _vec(rstd, M, "rstd"))
    return _call((_lib or load_library()).vcsr_layernorm, args, stream, timed)


def run_layernorm_grad_gpu(dy, s, weight, mean, rstd, dx, dweight=None, dbias=None, dsum=None,
                           workspace=None, stream=None, timed=False):
    """Gradients of run_layernorm_gpu (vcsr_layernorm_grad): s is the saved sum (x
    without a residual), dsum what flows into it from elsewhere; dx is the gradient of
    x and of the residual."""
    M, N = _shape2(s, "s")
    (dp, lddy), (sp, lds) = _mat(dy, M, N, "dy"), _mat(s, M, N, "s")
    (up, ldu), (xp, ldx) = _mat(dsum, M, N, "dsum", s.dtype), _mat(dx, M, N, "dx", s.dtype)
    xt, yt = _type(s, "s"), _type(dy, "dy")
    need = _layernorm_grad_bytes(M, N, xt, yt, dweight is not None, dbias is not None)
    args = _pack_layernorm_grad(M, N, xt, yt, dp, lddy, sp, lds, _vec(weight, N, "weight"),
                                _vec(mean, M, "mean"), _vec(rstd, M, "rstd"), up, ldu, xp, ldx,
                                _vec(dweight, N, "dweight"), _vec(dbias, N, "dbias"))
    return _call_with_space((_lib or load_library()).vcsr_layernorm_grad, args, need, workspace,
                            stream, timed)


def run_embed_gpu(table, ids, y, scale=1.0, table_scale=None, stream=None, timed=False):
    """y[m] = scale * table[ids[m]] (vcsr_embed).  table: float32, BF16, or FP8 with
    table_scale, one scale a row; ids: int32, those outside the table (padding) give rows
    of zeros; y: float32 or BF16."""
    (V, N), (ip, M) = _shape2(table, "table"), _ids(ids, "ids")
    (tp, ldt), (yp, ldy) = _mat(table, V, N, "table"), _mat(y, M, N, "y")
    args = _pack_embed(M, V, N, _type(table, "table"), _type(y, "y"), scale, tp, ldt,
                       _vec(table_scale, V, "table_scale"), ip, yp, ldy)
    return _call((_lib or load_library()).vcsr_embed, args, stream, timed)


def run_embed_grad_gpu(dy, ids, dtable, scale=1.0, accumulate=False, workspace=None, stream=None,
                       timed=False):
    """Gradient of run_embed_gpu (vcsr_embed_grad): dtable[v] = scale * the sum of dy's
    rows whose id is v, or that added to dtable's rows with accumulate.  dy, dtable:
    float32 or BF16."""
    (V, N), (ip, M) = _shape2(dtable, "dtable"), _ids(ids, "ids")
    (dp, lddy), (tp, lddt) = _mat(dy, M, N, "dy"), _mat(dtable, V, N, "dtable")
    tt, yt = _type(dtable, "dtable"), _type(dy, "dy")
    add = 1 if accumulate else 0
    need = _embed_grad_bytes(M, V, N, tt, yt, add)
    args = _pack_embed_grad(M, V, N, tt, yt, add, scale, dp, lddy, ip, tp, lddt)
    return _call_with_space((_lib or load_library()).vcsr_embed_grad, args, need, workspace, stream,
                            timed)


def _act(act):
    a = ACTIVATIONS.get(act)
    if a is None:
        raise VcsrError(VCSR_EINVAL, f"act: {act!r}, one of {sorted(ACTIVATIONS)} is expected")
    return a


def run_linear_gpu(x, w, y, bias=None, residual=None, act="none", z=None, x_scale=None,
                   w_scale=None, workspace=None, stream=None, timed=False):
    """y = act(x W^T + bias) + residual (vcsr_linear); w has one row per output
    column.  x, w: float32, BF16, or FP8 with x_scale and w_scale, one scale a
    row; y, z, residual: float32 or BF16.  z receives the activation's input."""
    (M, K), N = _shape2(x, "x"), _shape2(w, "w")[0]
    (xp, ldx), (wp, ldw) = _mat(x, M, K, "x"), _mat(w, N, K, "w", x.dtype)
    (yp, ldy), (rp, ldr) = _mat(y, M, N, "y"), _mat(residual, M, N, "residual", y.dtype)
    zp, ldz = _mat(z, M, N, "z", y.dtype)
    xt, yt = _type(x, "x"), _type(y, "y")
    args = _pack_linear(M, N, K, xt, yt, _act(act), xp, ldx, wp, ldw,
                        _vec(x_scale, M, "x_scale"), _vec(w_scale, N, "w_scale"),
                        _vec(bias, N, "bias"), rp, ldr, zp, ldz, yp, ldy)
    return _call_with_space((_lib or load_library()).vcsr_linear, args,
                            _linear_bytes(M, N, K, xt, yt, rp != 0, zp != 0), workspace, stream,
                            timed)


def run_linear_grad_gpu(dy, x, w, z=None, act="none", dx=None, dw=None, dbias=None,
                        workspace=None, stream=None, timed=False):
    """Gradients of run_linear_gpu (vcsr_linear_grad) from dy and the saved z
    (not needed for act "none"): those of dx, dw and dbias that are given.  The
    residual's gradient is dy."""
    (M, K), N = _shape2(x, "x"), _shape2(w, "w")[0]
    (xp, ldx), (wp, ldw) = _mat(x, M, K, "x"), _mat(w, N, K, "w", x.dtype)
    (dp, lddy), (zp, ldz) = _mat(dy, M, N, "dy"), _mat(z, M, N, "z", dy.dtype)
    (xg, lddx), (wg, lddw) = _mat(dx, M, K, "dx", x.dtype), _mat(dw, N, K, "dw", x.dtype)
    xt, yt, at = _type(x, "x"), _type(dy, "dy"), _act(act)
    need = _linear_grad_bytes(M, N, K, xt, yt, at, z is not None, dx is not None, dw is not None,
                              dbias is not None)
    args = _pack_linear_grad(M, N, K, xt, yt, at, dp, lddy, zp, ldz, xp, ldx, wp, ldw, xg, lddx,
                             wg, lddw, _vec(dbias, N, "dbias"))
    return _call_with_space((_lib or load_library()).vcsr_linear_grad, args, need, workspace,
                            stream, timed)


def _one_stride(a, b, what):
    if a is not None and b is not None and getattr(a, "ld", 0) != getattr(b, "ld", 0) and \
            getattr(a, "ld", a.shape[-1]) != getattr(b, "ld", b.shape[-1]):
        raise VcsrError(VCSR_EINVAL, f"{what}: row strides differ")


def run_gated_gpu(x, w_gate, w_up, y, gate_bias=None, up_bias=None, act="silu", z_gate=None,
                  z_up=None, x_scale=None, gate_scale=None, up_scale=None, workspace=None,
                  stream=None, timed=False):
    """y = act(x Wg^T + gate_bias) * (x Wu^T + up_bias) (vcsr_gated); the weights have one
    row per output column.  x, weights: float32, BF16, or FP8 with x_scale, gate_scale
    and up_scale, one scale a row; y, z_gate, z_up: float32 or BF16.  z_gate and z_up
    (both or neither, of one row stride) receive the two products."""
    (M, K), N = _shape2(x, "x"), _shape2(w_gate, "w_gate")[0]
    (xp, ldx), (gp, ldg) = _mat(x, M, K, "x"), _mat(w_gate, N, K, "w_gate", x.dtype)
    (up, ldu), (yp, ldy) = _mat(w_up, N, K, "w_up", x.dtype), _mat(y, M, N, "y")
    (zg, ldz), (zu, _) = _mat(z_gate, M, N, "z_gate", y.dtype), _mat(z_up, M, N, "z_up", y.dtype)
    _one_stride(z_gate, z_up, "z_gate, z_up")
    xt, yt = _type(x, "x"), _type(y, "y")
    args = _pack_gated(M, N, K, xt, yt, _act(act), xp, ldx, gp, ldg, up, ldu,
                       _vec(x_scale, M, "x_scale"), _vec(gate_scale, N, "gate_scale"),
                       _vec(up_scale, N, "up_scale"), _vec(gate_bias, N, "gate_bias"),
                       _vec(up_bias, N, "up_bias"), zg, zu, ldz, yp, ldy)
    return _call_with_space((_lib or load_library()).vcsr_gated, args,
                            _gated_bytes(M, N, K, xt, yt, zg != 0), workspace, stream, timed)


def run_gated_grad_gpu(dy, x, w_gate, w_up, z_gate, z_up, act="silu", dx=None, dw_gate=None,
                       dw_up=None, dgate_bias=None, dup_bias=None, workspace=None, stream=None,
                       timed=False):
    """Gradients of run_gated_gpu (vcsr_gated_grad) from dy and the saved z_gate and z_up:
    those of dx, dw_gate with dw_up, dgate_bias and dup_bias that are given."""
    (M, K), N = _shape2(x, "x"), _shape2(w_gate, "w_gate")[0]
    (xp, ldx), (gp, ldg) = _mat(x, M, K, "x"), _mat(w_gate, N, K, "w_gate", x.dtype)
    (up, ldu), (dp, lddy) = _mat(w_up, N, K, "w_up", x.dtype), _mat(dy, M, N, "dy")
    (zg, ldz), (zu, _) = _mat(z_gate, M, N, "z_gate", dy.dtype), _mat(z_up, M, N, "z_up", dy.dtype)
    _one_stride(z_gate, z_up, "z_gate, z_up")
    (xg, lddx), (gg, lddg) = _mat(dx, M, K, "dx", x.dtype), _mat(dw_gate, N, K, "dw_gate", x.dtype)
    ug, lddu = _mat(dw_up, N, K, "dw_up", x.dtype)
    xt, yt = _type(x, "x"), _type(dy, "dy")
    need = _gated_grad_bytes(M, N, K, xt, yt, dx is not None, dw_gate is not None,
                             dgate_bias is not None, dup_bias is not None)
    args = _pack_gated_grad(M, N, K, xt, yt, _act(act), dp, lddy, zg, zu, ldz, xp, ldx, gp, ldg, up,
                            ldu, xg, lddx, gg, lddg, ug, lddu,
                            _vec(dgate_bias, N, "dgate_bias"), _vec(dup_bias, N, "dup_bias"))
    return _call_with_space((_lib or load_library()).vcsr_gated_grad, args, need, workspace, stream,
                            timed)


class AdamW:
    """One AdamW step over all tensors of a model (vcsr_adamw_create / _step).

    `tensors`: dicts of device buffers `param` (float32), `grad` (float32 or
    BF16), `m` and `v` (float32, or FP8 with `m_scale` and `v_scale`, one
    float32 per 256 values), optionally `copy` (BF16, receives the parameter)
    and a number `weight_decay`.  Zeroed states start a run."""

    def __init__(self, tensors, stream=None):
        table = (_AdamwTensor * max(len(tensors), 1))()
        for i, t in enumerate(tensors):
            n = int(np.prod(t["param"].shape))
            fp8 = t["m"].dtype == FP8
            blocks = -(-n // 256)
            for name, dtypes, count in (("param", (F32,), n), ("grad", (F32, BF16), n),
                                        ("m", (F32, FP8), n), ("v", (t["m"].dtype,), n),
                                        ("m_scale", (F32,), blocks), ("v_scale", (F32,), blocks),
                                        ("copy", (BF16,), n)):
                b = t.get(name)
                if b is None:
                    if name == "copy" or (not fp8 and name in ("m_scale", "v_scale")):
                        continue
                    raise VcsrError(VCSR_EINVAL, f"tensor {i}: {name} is missing")
                if b.dtype not in dtypes or b.nbytes < count * b.dtype.itemsize or \
                        getattr(b, "ld", b.shape[-1] if b.shape else 1) != \
                        (b.shape[-1] if b.shape else 1):
                    raise VcsrError(VCSR_EINVAL, f"tensor {i}: {name}: {b.dtype}, {b.nbytes} "
                                                 f"bytes; {count} contiguous values are expected")
            ptr = {k: t[k].ptr if t.get(k) is not None else None for k in
                   ("param", "grad", "m", "v", "m_scale", "v_scale", "copy")}
            table[i] = _AdamwTensor(n, _TYPE[t["grad"].dtype], _TYPE[t["m"].dtype], ptr["param"],
                                    ptr["grad"], ptr["m"], ptr["v"], ptr["m_scale"],
                                    ptr["v_scale"], ptr["copy"], t.get("weight_decay", 0.0))
        self._keep = [dict(t) for t in tensors]
        self._h = C.c_void_p()
        _check(load_library().vcsr_adamw_create(table, len(tensors), _sp(stream),
                                                C.byref(self._h)))

    def step(self, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, stream=None,
             timed=False):
        """The step numbered `step` (1 for the first); gradients are multiplied
        by grad_scale first.  Enqueued only, unless timed."""
        ms = C.c_float(0)
        hyper = _AdamwHyper(lr, beta1, beta2, eps, grad_scale, step)
        _check(load_library().vcsr_adamw_step(self._h, C.byref(hyper), _sp(stream),
                                              C.byref(ms) if timed else None))
        return ms.value if timed else None

    def __del__(self):
        if getattr(self, "_h", None) and _lib is not None and self._h.value:
            _lib.vcsr_adamw_free(self._h)
            self._h = C.c_void_p()
