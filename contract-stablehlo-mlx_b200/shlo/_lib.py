"""ctypes binding of libshlo_cuda.so (include/shlo_cuda.h)."""
from __future__ import annotations

import ctypes
import os
import struct

PKG = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.environ.get("SHLO_CUDA_LIB", os.path.join(PKG, "lib", "libshlo_cuda.so"))

# Every exported symbol of include/shlo_cuda.h.
SYMBOLS = [
    "shlo_last_error", "shlo_set_device", "shlo_get_device", "shlo_device_count", "shlo_set_flavor",
    "shlo_get_flavor", "shlo_retain", "shlo_release", "shlo_empty", "shlo_of_bytes", "shlo_nbytes",
    "shlo_to_bytes", "shlo_shape", "shlo_dtype", "shlo_unary", "shlo_binary", "shlo_where", "shlo_reshape",
    "shlo_transpose", "shlo_broadcast", "shlo_slice", "shlo_concat", "shlo_astype", "shlo_view", "shlo_take",
    "shlo_max_axis", "shlo_contiguous", "shlo_eval", "shlo_kernel_new", "shlo_kernel_free",
    "shlo_kernel_apply", "shlo_compile", "shlo_fn_free", "shlo_apply", "shlo_libm_erff_range",
    "shlo_count_nonzero", "shlo_current_stream", "shlo_launch_count", "shlo_device_ptr", "shlo_mul_mat_noalloc",
    "shlo_rope_phases", "shlo_rope_noalloc", "shlo_kv_append_noalloc", "shlo_kv_gather_noalloc",
    "shlo_cuda_device", "shlo_kv_attend_workspace", "shlo_kv_attend_noalloc",
    "shlo_kv_new", "shlo_kv_free", "shlo_kv_storage", "shlo_kv_append", "shlo_kv_gather", "shlo_kv_attend",
    "shlo_test_attend_give_up",
    "shlo_norm_rope_noalloc", "shlo_norm_rope_workspace", "shlo_norm_rope_grad_noalloc", "shlo_quantise_rows_noalloc",
    "shlo_mul_mat8_noalloc", "shlo_linear8_workspace", "shlo_linear8_noalloc", "shlo_beam_workspace",
    "shlo_beam_select_noalloc", "shlo_kv_fork_noalloc", "shlo_kv_fork", "shlo_norm_rope_grad", "shlo_quantise_rows",
    "shlo_linear8", "shlo_beam_select",
]


class ShloError(RuntimeError):
    """An error status from libshlo_cuda (the message of shlo_last_error)."""


c_arr = ctypes.c_void_p
c_i64p = ctypes.POINTER(ctypes.c_int64)
TRACE_FN = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, ctypes.POINTER(c_arr), ctypes.c_int,
                            ctypes.POINTER(c_arr), ctypes.POINTER(ctypes.c_int), ctypes.c_int,
                            ctypes.c_void_p, ctypes.c_size_t)
FREE_FN = ctypes.CFUNCTYPE(None, ctypes.c_void_p)



class KvPool(ctypes.Structure):
    """shlo_kv_pool."""
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("k_scale", ctypes.c_void_p),
                ("v_scale", ctypes.c_void_p), ("pages", ctypes.c_int64), ("page_stride", ctypes.c_int64),
                ("head_stride", ctypes.c_int64), ("token_stride", ctypes.c_int64),
                ("scale_page_stride", ctypes.c_int64), ("scale_head_stride", ctypes.c_int64),
                ("heads", ctypes.c_int32), ("head_dim", ctypes.c_int32), ("page_tokens", ctypes.c_int32)]


class KvBatch(ctypes.Structure):
    """shlo_kv_batch."""
    _fields_ = [("starts", ctypes.c_void_p), ("lens", ctypes.c_void_p), ("tables", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("seqs", ctypes.c_int32), ("table_pages", ctypes.c_int32),
                ("tokens", ctypes.c_int32)]


# The descriptors of include/shlo_cuda.h that a call fills anew, in their fields' order (native alignment).
NORM_ROPE_ARGS = struct.Struct("PqqPPPPPqqPqqPPPNqiiiiffIBB")
MUL_MAT8_ARGS = struct.Struct("PqPPqPPPqPNqiiBB")
BEAM_ARGS = struct.Struct("PqPPPPPPNiiiiiB")
KV_FORK_ARGS = struct.Struct("PPqPPPPqiii")

_lib = None


def load() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError("libshlo_cuda.so is not built (%s); run contract-stablehlo-mlx_b200/build.py" % LIB_PATH)
    L = ctypes.CDLL(LIB_PATH)
    i = ctypes.c_int
    L.shlo_last_error.restype = ctypes.c_char_p
    L.shlo_last_error.argtypes = []
    L.shlo_set_device.argtypes = [i]
    L.shlo_get_device.argtypes = [ctypes.POINTER(i)]
    L.shlo_device_count.argtypes = [ctypes.POINTER(i)]
    L.shlo_set_flavor.argtypes = [i]
    L.shlo_get_flavor.argtypes = [ctypes.POINTER(i)]
    L.shlo_retain.argtypes = [c_arr]
    L.shlo_retain.restype = None
    L.shlo_release.argtypes = [c_arr]
    L.shlo_release.restype = None
    L.shlo_empty.argtypes = []
    L.shlo_empty.restype = c_arr
    L.shlo_of_bytes.argtypes = [ctypes.c_void_p, ctypes.c_size_t, c_i64p, i, ctypes.c_uint8, ctypes.POINTER(c_arr)]
    L.shlo_nbytes.argtypes = [c_arr, ctypes.POINTER(ctypes.c_size_t)]
    L.shlo_to_bytes.argtypes = [c_arr, ctypes.c_void_p, ctypes.c_size_t]
    L.shlo_shape.argtypes = [c_arr, c_i64p, ctypes.POINTER(i)]
    L.shlo_dtype.argtypes = [c_arr, ctypes.POINTER(ctypes.c_uint8)]
    L.shlo_unary.argtypes = [ctypes.c_uint32, c_arr, ctypes.POINTER(c_arr)]
    L.shlo_binary.argtypes = [ctypes.c_uint32, c_arr, c_arr, ctypes.POINTER(c_arr)]
    L.shlo_where.argtypes = [c_arr, c_arr, c_arr, ctypes.POINTER(c_arr)]
    L.shlo_reshape.argtypes = [c_arr, c_i64p, i, ctypes.POINTER(c_arr)]
    L.shlo_transpose.argtypes = [c_arr, c_i64p, i, ctypes.POINTER(c_arr)]
    L.shlo_broadcast.argtypes = [c_arr, c_i64p, i, ctypes.POINTER(c_arr)]
    L.shlo_slice.argtypes = [c_arr, c_i64p, c_i64p, c_i64p, i, ctypes.POINTER(c_arr)]
    L.shlo_concat.argtypes = [ctypes.POINTER(c_arr), i, ctypes.c_uint32, ctypes.POINTER(c_arr)]
    L.shlo_astype.argtypes = [c_arr, ctypes.c_uint8, ctypes.POINTER(c_arr)]
    L.shlo_view.argtypes = [c_arr, ctypes.c_uint8, ctypes.POINTER(c_arr)]
    L.shlo_take.argtypes = [c_arr, c_arr, ctypes.c_uint32, ctypes.POINTER(c_arr)]
    L.shlo_max_axis.argtypes = [c_arr, ctypes.c_uint32, ctypes.POINTER(c_arr)]
    L.shlo_contiguous.argtypes = [c_arr, ctypes.POINTER(c_arr)]
    L.shlo_eval.argtypes = [ctypes.POINTER(c_arr), i]
    L.shlo_kernel_new.argtypes = [ctypes.c_char_p, ctypes.POINTER(ctypes.c_char_p), i,
                                  ctypes.POINTER(ctypes.c_char_p), i, ctypes.c_char_p, ctypes.c_char_p,
                                  ctypes.POINTER(ctypes.c_void_p)]
    L.shlo_kernel_free.argtypes = [ctypes.c_void_p]
    L.shlo_kernel_free.restype = None
    L.shlo_kernel_apply.argtypes = [ctypes.c_void_p, ctypes.POINTER(c_arr), i, ctypes.POINTER(c_i64p),
                                    ctypes.POINTER(i), ctypes.POINTER(ctypes.c_uint8), i, c_i64p, c_i64p,
                                    ctypes.POINTER(c_arr)]
    L.shlo_compile.argtypes = [TRACE_FN, ctypes.c_void_p, FREE_FN, i, ctypes.POINTER(ctypes.c_void_p)]
    L.shlo_fn_free.argtypes = [ctypes.c_void_p]
    L.shlo_fn_free.restype = None
    L.shlo_apply.argtypes = [ctypes.c_void_p, ctypes.POINTER(c_arr), i, ctypes.POINTER(c_arr),
                             ctypes.POINTER(i), i]
    L.shlo_libm_erff_range.argtypes = [ctypes.c_uint32, ctypes.c_uint32, ctypes.c_void_p]
    L.shlo_count_nonzero.argtypes = [c_arr, ctypes.POINTER(ctypes.c_uint64)]
    L.shlo_current_stream.argtypes = [ctypes.POINTER(ctypes.c_void_p)]
    L.shlo_launch_count.argtypes = [ctypes.POINTER(ctypes.c_uint64)]
    L.shlo_device_ptr.argtypes = [c_arr, ctypes.POINTER(ctypes.c_void_p), ctypes.POINTER(i)]
    L.shlo_mul_mat_noalloc.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64,
                                       ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
                                       ctypes.c_void_p]
    p, i32, i64, u8 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_uint8
    f32, f64 = ctypes.c_float, ctypes.c_double
    pool, batch = ctypes.POINTER(KvPool), ctypes.POINTER(KvBatch)
    L.shlo_rope_phases.argtypes = [i32, f64, i32, f64, f64, f64, f64, p, ctypes.POINTER(f32)]
    L.shlo_rope_noalloc.argtypes = [p, i64, i64, p, p, p, i64, i64, i64, i32, i32, i32, u8, ctypes.c_uint32, f32, p]
    L.shlo_kv_append_noalloc.argtypes = [pool, batch, p, i64, i64, p, i64, i64, u8, p]
    L.shlo_kv_gather_noalloc.argtypes = [pool, p, i64, i32, i32, p, p, i64, p, i64, i64, p, i64, i64, u8, p]
    L.shlo_cuda_device.argtypes = []
    u32, size, sizep = ctypes.c_uint32, ctypes.c_size_t, ctypes.POINTER(ctypes.c_size_t)
    packed = ctypes.c_char_p  # (a descriptor's bytes: one conversion a call, where fields as arguments take one each)
    for name in ("norm_rope", "norm_rope_grad", "mul_mat8", "linear8", "beam_select"):
        getattr(L, "shlo_%s_noalloc" % name).argtypes = [packed, p]
    L.shlo_norm_rope_workspace.argtypes = [sizep]
    L.shlo_quantise_rows_noalloc.argtypes = [p, i64, i64, i32, u8, p, i64, p, p]
    L.shlo_linear8_workspace.argtypes = [i64, i32, sizep]
    L.shlo_beam_workspace.argtypes = [i32, i32, i32, i32, sizep]
    L.shlo_kv_fork_noalloc.argtypes = [pool, packed, p]
    L.shlo_kv_attend_workspace.argtypes = [ctypes.POINTER(ctypes.c_size_t)]
    L.shlo_kv_attend_noalloc.argtypes = [pool, batch, p, i64, i64, i32, u8, f32, i32, i32, p, i64, i64, p, p,
                                         ctypes.c_size_t, p]
    outp = ctypes.POINTER(p)
    L.shlo_kv_fork.argtypes = [p, c_arr, c_arr, c_arr, c_arr, outp, outp]
    L.shlo_norm_rope_grad.argtypes = [c_arr] * 6 + [i32, f32, u32, f32, outp, outp, outp]
    L.shlo_quantise_rows.argtypes = [c_arr, outp, outp]
    L.shlo_linear8.argtypes = [c_arr, c_arr, c_arr, c_arr, c_arr, u8, outp]
    L.shlo_beam_select.argtypes = [c_arr, c_arr, c_arr, i32, i32, outp, outp, outp]
    L.shlo_kv_new.argtypes = [i64, i32, i32, i32, ctypes.POINTER(p)]
    L.shlo_kv_free.argtypes = [p]
    L.shlo_kv_free.restype = None
    L.shlo_kv_storage.argtypes = [p, pool]
    L.shlo_kv_append.argtypes = [p, c_arr, c_arr, c_arr, c_arr, c_arr]
    L.shlo_kv_gather.argtypes = [p, c_arr, c_arr, c_arr, u8, ctypes.POINTER(c_arr), ctypes.POINTER(c_arr)]
    L.shlo_kv_attend.argtypes = [p, c_arr, c_arr, c_arr, c_arr, f32, i32, i32, ctypes.POINTER(c_arr),
                                 ctypes.POINTER(c_arr)]
    L.shlo_test_attend_give_up.argtypes = [i32]
    L.shlo_test_attend_give_up.restype = None
    special = {"shlo_last_error", "shlo_empty", "shlo_retain", "shlo_release", "shlo_kernel_free", "shlo_fn_free",
               "shlo_kv_free", "shlo_test_attend_give_up"}
    for name in SYMBOLS:
        if name not in special:
            getattr(L, name).restype = ctypes.c_int
    _lib = L
    return L


def check(rc: int) -> None:
    if rc != 0:
        raise ShloError(load().shlo_last_error().decode("utf-8", "replace"))
