"""ctypes binding of libb200q.so (the C ABI in include/b200q.h).

The library is loaded from the package directory.  There is no fallback: if the shared
library is missing or fails to load, importing an op raises, so a GPU run can never silently
use anything but the CUDA kernels.
"""
from __future__ import annotations

import ctypes
import struct
from ctypes import POINTER, Structure, c_int, c_int8, c_int32, c_int64, c_longlong, c_size_t, c_uint8
from ctypes import c_uint64, c_void_p, c_float, c_char_p
from pathlib import Path

LIB_PATH = Path(__file__).resolve().parent / "libb200q.so"

B200Q_OK = 0
B200Q_ERR_INVALID_ARG = 1
B200Q_ERR_UNSUPPORTED = 2
B200Q_ERR_CUDA = 3
B200Q_ERR_TIMEOUT = 4

OUT_S32, OUT_S8, OUT_F32 = 0, 1, 2

PATH_NAMES = {
    0: "none",
    1: "tcgen05-im2col",
    2: "tcgen05-tiled",
    3: "cuda-core-generic",
    4: "cuda-core-depthwise",
    5: "cuda-core-qi32",
    6: "cuda-core-bmm-i32",
    7: "tcgen05-packed",
    8: "tcgen05-tiled-2sm",
    9: "tcgen05-rowtile",
    10: "tcgen05-s2d",
    11: "tcgen05-qi32",
    12: "cuda-core-depthwise-tma",
    13: "tcgen05-f32",
    14: "cuda-core-f32",
    15: "tcgen05-tiled-grouped",
    16: "tcgen05-bmm-i32",
    17: "linear-w4",
    18: "qk-norm-rope",
    19: "kv4-cache",
    20: "kv4-attention",
    21: "rows-s8",
    22: "linear-s8",
    23: "tcgen05-prompt-attention",
    24: "mma-prompt-attention",
}


class CConvParams(Structure):
    """Same layout as Conv2DParams (src/conv_types.h:21-29)."""

    _fields_ = [("pad_h", c_int), ("pad_w", c_int), ("stride_h", c_int), ("stride_w", c_int),
                ("dilation_h", c_int), ("dilation_w", c_int), ("groups", c_int)]


class CEpilogue(Structure):
    _fields_ = [("out_kind", c_int), ("zp_out", c_int), ("clamp_lo", c_int), ("clamp_hi", c_int)]


class CKV4Cache(Structure):
    _fields_ = [("k_codes", c_void_p), ("k_params", c_void_p), ("v_codes", c_void_p), ("v_params", c_void_p),
                ("pages", c_int), ("heads", c_int), ("page_size", c_int), ("d", c_int), ("group", c_int)]


class CLinearW4Args(Structure):
    _fields_ = [("x", c_void_p), ("ldx", c_int64), ("codes", c_void_p), ("scales", c_void_p), ("zeros", c_void_p),
                ("bias", c_void_p), ("y", c_void_p), ("ldy", c_int64), ("ftype", c_int), ("m", c_int), ("n", c_int),
                ("k", c_int), ("group", c_int)]


class CQKNormArgs(Structure):
    _fields_ = [(f, c_void_p) for f in ("q", "k", "q_w", "k_w", "table", "pos", "q_out", "k_out", "q_grad", "k_grad",
                                        "q_w_grad", "k_w_grad")]
    _fields_ += [(f, c_int64) for f in ("q_ts", "q_hs", "k_ts", "k_hs", "qo_ts", "qo_hs", "ko_ts", "ko_hs")]
    _fields_ += [(f, c_int) for f in ("positions", "ftype", "t", "hq", "hk", "d", "rot", "interleaved")]
    _fields_ += [("eps", c_float)]


class CKV4AttentionArgs(Structure):
    _fields_ = [("q", c_void_p), ("q_bs", c_int64), ("q_ts", c_int64), ("q_hs", c_int64), ("block_table", c_void_p),
                ("bt_stride", c_int64), ("lens", c_void_p), ("out", c_void_p), ("lse", c_void_p), ("ftype", c_int),
                ("b", c_int), ("tq", c_int), ("hq", c_int), ("max_pages", c_int), ("scale", c_float)]


class CRowsS8Args(Structure):
    _fields_ = [("x", c_void_p), ("ldx", c_int64), ("w", c_void_p), ("residual", c_void_p), ("ldr", c_int64),
                ("sum", c_void_p), ("lds", c_int64), ("codes", c_void_p), ("ldc", c_int64), ("scales", c_void_p),
                ("ftype", c_int), ("t", c_int), ("n", c_int), ("eps", c_float)]


class CReadS8Args(Structure):
    _fields_ = [("codes", c_void_p), ("ldc", c_int64), ("scales", c_void_p), ("y", c_void_p), ("ldy", c_int64),
                ("ftype", c_int), ("t", c_int), ("n", c_int)]


class CLinearS8Args(Structure):
    _fields_ = [("x", c_void_p), ("ldx", c_int64), ("x_scales", c_void_p), ("w", c_void_p), ("ldw", c_int64),
                ("w_scales", c_void_p), ("bias", c_void_p), ("y", c_void_p), ("ldy", c_int64), ("ftype", c_int),
                ("m", c_int), ("n", c_int), ("k", c_int)]


class CPromptAttentionArgs(Structure):
    _fields_ = [("q", c_void_p), ("q_ts", c_int64), ("q_hs", c_int64), ("k", c_void_p), ("k_ts", c_int64),
                ("k_hs", c_int64), ("v", c_void_p), ("v_ts", c_int64), ("v_hs", c_int64), ("starts", c_void_p),
                ("k_starts", c_void_p), ("out", c_void_p), ("lse", c_void_p)]
    _fields_ += [(f, c_int) for f in ("ftype", "b", "tq", "tk", "hq", "hk", "d")]
    _fields_ += [("scale", c_float)]


def packer(layout) -> "struct.Struct":
    """The bytes of a ctypes structure's fields in order: an argument block is packed and handed over in a fraction
    of the time that filling the structure takes."""
    code = {c_void_p: "P", c_int64: "q", c_int: "i", c_float: "f"}
    fmt = "".join(code[t] for _, t in layout._fields_)
    return struct.Struct(fmt + "x" * (ctypes.sizeof(layout) - struct.calcsize(fmt)))


class B200QError(RuntimeError):
    """Raised for a non-zero status; ``code`` is the b200q_status value."""

    def __init__(self, code: int, msg: str):
        super().__init__(msg)
        self.code = code


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise RuntimeError(f"{LIB_PATH} is not built; run __graft_entry__.build() "
                           "(the CUDA library is required, there is no CPU path)")
    L = ctypes.CDLL(str(LIB_PATH))
    vp, i, ll = c_void_p, c_int, c_longlong
    pconv, pepi, packed = POINTER(CConvParams), POINTER(CEpilogue), c_char_p
    sig = {
        "b200q_fprop_nhwc_qi32": [i, vp, vp, vp, i, i, i, i, i, i, i, pconv, vp, vp, vp],
        "b200q_block_fprop_nhwc_qi32": [i, vp, vp, vp, i, i, i, i, i, i, i, pconv, i, i, vp, vp, vp],
        "b200q_bmm_matmul_i32": [vp, vp, vp, i, i, i, i, i, i, vp],
        "b200q_conv2d_s8": [vp, vp, vp, vp, vp, i, i, i, i, i, i, i, pconv, pepi, vp],
        "b200q_conv2d_s8_packed_noalloc": [vp, vp, vp, vp, vp, i, i, i, i, i, i, i, pconv, pepi, vp],
        "b200q_conv2d_s8_add": [vp, vp, vp, vp, vp, c_float, vp, i, i, i, i, i, i, i, pconv, pepi, vp],
        "b200q_maxpool_s8": [vp, vp, i, i, i, i, i, i, i, i, i, i, vp],
        "b200q_global_avgpool_s8": [vp, vp, i, i, i, i, vp],
        "b200q_bmm_s8": [vp, vp, vp, vp, vp, i, i, i, i, i, i, pepi, vp],
        "b200q_conv_out_shape": [i, i, i, i, i, i, pconv, POINTER(c_int), POINTER(c_int)],
        "b200q_conv2d_s8_plan": [i, i, i, i, i, i, i, pconv, pepi, i, POINTER(c_int)],
        "b200q_device_error": [],
        "b200q_last_path": [],
        "b200q_fill_s8_uniform": [vp, c_size_t, c_uint64, c_uint64, i, i, vp],
        "b200q_fill_i32_uniform": [vp, c_size_t, c_uint64, c_uint64, c_int32, c_int32, vp],
        "b200q_fill_s8_table": [vp, c_size_t, c_uint64, c_uint64, vp, vp],
        "b200q_selftest_wait_timeout": [c_longlong],
        "b200q_conv_fprop_f32": [vp, vp, vp, i, vp, i, i, i, i, i, i, i, pconv, i, i, vp],
        "b200q_conv_bprop_f32": [vp, vp, vp, i, i, i, i, i, i, i, pconv, i, i, vp],
        "b200q_conv_grad_f32": [vp, vp, vp, vp, i, i, i, i, i, i, i, i, pconv, i, i, vp],
        "b200q_bmm_f32": [vp, vp, vp, i, i, i, i, i, i, vp],
        "b200q_linear_w4": [packed, vp],
        "b200q_qk_norm_rope": [packed, vp],
        "b200q_qk_norm_rope_bprop": [packed, vp],
        "b200q_kv4_append": [packed, vp, ll, ll, vp, ll, ll, vp, i, i, vp],
        "b200q_kv4_read": [packed, vp, vp, vp, i, i, vp],
        "b200q_kv4_attention": [packed, packed, vp],
        "b200q_quantize_s8": [packed, vp],
        "b200q_rms_norm_s8": [packed, vp],
        "b200q_read_s8": [packed, vp],
        "b200q_linear_s8": [packed, vp],
        "b200q_prompt_attention": [packed, vp],
    }
    for name, args in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = c_int
    L.b200q_last_error.argtypes = []
    L.b200q_last_error.restype = c_char_p
    L.b200q_set_path_policy.argtypes = [c_int]
    L.b200q_set_path_policy.restype = None
    L.b200q_noalloc_scratch_bytes.argtypes = []
    L.b200q_noalloc_scratch_bytes.restype = c_size_t
    L.b200q_tc_launch_count.argtypes = []
    L.b200q_tc_launch_count.restype = c_longlong
    _lib = L
    return L


def check(rc: int) -> None:
    if rc != B200Q_OK:
        msg = lib().b200q_last_error().decode(errors="replace")
        raise B200QError(rc, msg)


def device_error() -> None:
    """Synchronizes the device and raises B200QError for what its error word holds (see
    b200q_device_error): a wait that ran out, or a position, slot, page or length out of range."""
    check(lib().b200q_device_error())


def last_path() -> str:
    return PATH_NAMES.get(lib().b200q_last_path(), "?")


def set_path_policy(policy: int) -> None:
    lib().b200q_set_path_policy(policy)


def tc_launch_count() -> int:
    return int(lib().b200q_tc_launch_count())


EXPORTED_SYMBOLS = [
    "b200q_fprop_nhwc_qi32", "b200q_block_fprop_nhwc_qi32", "b200q_bmm_matmul_i32",
    "b200q_conv2d_s8", "b200q_bmm_s8", "b200q_conv_out_shape", "b200q_last_error",
    "b200q_device_error", "b200q_last_path", "b200q_set_path_policy", "b200q_tc_launch_count",
    "b200q_fill_s8_uniform", "b200q_fill_i32_uniform", "b200q_fill_s8_table",
    "b200q_selftest_wait_timeout", "b200q_conv2d_s8_packed_noalloc", "b200q_noalloc_scratch_bytes",
    "b200q_conv_fprop_f32", "b200q_conv_bprop_f32", "b200q_conv_grad_f32", "b200q_bmm_f32",
    "b200q_conv2d_s8_add", "b200q_maxpool_s8", "b200q_global_avgpool_s8", "b200q_conv2d_s8_plan",
    "b200q_linear_w4", "b200q_qk_norm_rope", "b200q_qk_norm_rope_bprop", "b200q_kv4_append", "b200q_kv4_read",
    "b200q_kv4_attention", "b200q_quantize_s8", "b200q_rms_norm_s8", "b200q_read_s8", "b200q_linear_s8",
    "b200q_prompt_attention",
]
