"""ctypes bindings of the C ABI in include/ogle_cuda.h.

The library is the product: if libogle_cuda.so is missing this module raises,
it never falls back to another implementation.
"""
import ctypes as C
import os
import struct

_HERE = os.path.dirname(os.path.abspath(__file__))
CUDA_LIB_PATH = os.path.join(_HERE, "libogle_cuda.so")
RT_LIB_PATH = os.path.join(_HERE, "libogle_rt.so")

OGLE_MAX_CONCAT_INPUTS = 16

MATH_FP32, MATH_TF32, MATH_TF32X3 = 0, 1, 2
ATTENTION_NO_WORKSPACE = 64
DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2
ACT_NONE, ACT_CLIP, ACT_RELU = 0, 1, 2


class ConvParams(C.Structure):
    _fields_ = [
        ("N", C.c_int), ("in_hwc", C.c_int * 3), ("out_hwc", C.c_int * 3),
        ("kernel", C.c_int), ("stride", C.c_int), ("pad", C.c_int), ("dilation", C.c_int), ("group", C.c_int),
        ("has_bias", C.c_int), ("act", C.c_int), ("min_value", C.c_float), ("max_value", C.c_float),
        ("in_channel_stride", C.c_int), ("out_channel_stride", C.c_int), ("out_channel_offset", C.c_int),
        ("math_mode", C.c_int), ("n_tile", C.c_int), ("split", C.c_int), ("channels_on_m", C.c_int), ("sm_pair", C.c_int),
    ]


class PoolParams(C.Structure):
    _fields_ = [
        ("N", C.c_int), ("in_hwc", C.c_int * 3), ("out_hwc", C.c_int * 3),
        ("kernel", C.c_int), ("stride", C.c_int), ("pad", C.c_int), ("type", C.c_int),
        ("in_channel_stride", C.c_int), ("out_channel_stride", C.c_int),
    ]


class GemmParams(C.Structure):
    _fields_ = [
        ("M", C.c_int), ("K", C.c_int), ("N", C.c_int), ("transB", C.c_int),
        ("alpha", C.c_float), ("beta", C.c_float), ("bias_mode", C.c_int),
        ("lda", C.c_int), ("ldb", C.c_int), ("ldc", C.c_int), ("ldy", C.c_int), ("math_mode", C.c_int),
    ]


class ConcatParams(C.Structure):
    _fields_ = [("n_inputs", C.c_int), ("axis", C.c_int), ("in_shapes", (C.c_int * 4) * OGLE_MAX_CONCAT_INPUTS)]


class Contraction(C.Structure):
    _fields_ = [("form", C.c_int), ("ranges", C.c_int), ("n_tile", C.c_int), ("overlapped", C.c_int)]


class DetectParams(C.Structure):
    _fields_ = [
        ("N", C.c_int), ("A", C.c_int), ("C", C.c_int), ("logit_stride", C.c_int), ("mode", C.c_int),
        ("score_thr", C.c_float), ("top_k", C.c_int), ("nms_thr", C.c_float),
        ("image_w", C.c_int), ("image_h", C.c_int), ("frame_sizes", C.c_void_p),
    ]


class PagedBatch(C.Structure):
    _fields_ = [
        ("n_seqs", C.c_int), ("n_rows", C.c_int), ("max_rows", C.c_int), ("max_kv_len", C.c_int),
        ("q_heads", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int), ("page_tokens", C.c_int),
        ("n_pages", C.c_int), ("table_stride", C.c_int), ("dtype", C.c_int), ("reserved", C.c_int),
        ("page_stride", C.c_longlong), ("head_stride", C.c_longlong), ("token_stride", C.c_longlong),
        ("row_start", C.c_void_p), ("kv_len", C.c_void_p), ("block_table", C.c_void_p),
        ("k_cache", C.c_void_p), ("v_cache", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
    ]


class AppendParams(C.Structure):
    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("q", C.c_void_p), ("q_out", C.c_void_p),
        ("k_row", C.c_longlong), ("k_head", C.c_longlong), ("v_row", C.c_longlong), ("v_head", C.c_longlong),
        ("q_row", C.c_longlong), ("q_head", C.c_longlong), ("q_out_row", C.c_longlong), ("q_out_head", C.c_longlong),
        ("rotary", C.c_void_p), ("rotary_dim", C.c_int), ("rotary_rows", C.c_int), ("interleaved", C.c_int),
        ("reserved", C.c_int),
    ]


class AttentionParams(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("out", C.c_void_p), ("lse", C.c_void_p),
        ("q_row", C.c_longlong), ("q_head", C.c_longlong), ("out_row", C.c_longlong), ("out_head", C.c_longlong),
        ("scale", C.c_float), ("causal", C.c_int), ("window", C.c_int), ("reserved", C.c_int),
    ]


class LogitsParams(C.Structure):
    _fields_ = [
        ("rows", C.c_int), ("vocab", C.c_int), ("dtype", C.c_int), ("out_dtype", C.c_int),
        ("n_tokens", C.c_int), ("n_biases", C.c_int),
        ("logits_stride", C.c_longlong), ("out_stride", C.c_longlong), ("allowed_stride", C.c_longlong),
        ("logits", C.c_void_p), ("out", C.c_void_p),
        ("tokens", C.c_void_p), ("token_start", C.c_void_p), ("prompt_len", C.c_void_p),
        ("repetition", C.c_void_p), ("presence", C.c_void_p), ("frequency", C.c_void_p),
        ("bias_token", C.c_void_p), ("bias_value", C.c_void_p), ("bias_start", C.c_void_p), ("allowed", C.c_void_p),
    ]


class BeamParams(C.Structure):
    _fields_ = [
        ("n_groups", C.c_int), ("beams", C.c_int), ("vocab", C.c_int), ("count", C.c_int), ("dtype", C.c_int), ("n_ends", C.c_int),
        ("logits_stride", C.c_longlong), ("logits", C.c_void_p), ("scores", C.c_void_p), ("ends", C.c_void_p),
        ("out_score", C.c_void_p), ("out_beam", C.c_void_p), ("out_token", C.c_void_p),
        ("next_row", C.c_void_p), ("next_token", C.c_void_p), ("next_score", C.c_void_p),
    ]


class AdvanceParams(C.Structure):
    _fields_ = [
        ("n_old", C.c_int), ("n_new", C.c_int), ("old_blocks", C.c_int), ("new_blocks", C.c_int),
        ("page_tokens", C.c_int), ("n_pages", C.c_int), ("new_tokens", C.c_int), ("reserved", C.c_int),
        ("old_stride", C.c_longlong), ("new_stride", C.c_longlong),
        ("table", C.c_void_p), ("kv_len", C.c_void_p), ("parent", C.c_void_p), ("tokens", C.c_void_p), ("refs", C.c_void_p),
        ("new_table", C.c_void_p), ("new_len", C.c_void_p), ("new_refs", C.c_void_p), ("copies", C.c_void_p), ("state", C.c_void_p),
    ]


class CompactParams(C.Structure):
    _fields_ = [
        ("n_seqs", C.c_int), ("blocks", C.c_int), ("page_tokens", C.c_int), ("n_pages", C.c_int), ("n_copies", C.c_int), ("reserved", C.c_int),
        ("table_stride", C.c_longlong), ("new_stride", C.c_longlong),
        ("table", C.c_void_p), ("refs", C.c_void_p), ("new_table", C.c_void_p), ("new_refs", C.c_void_p),
        ("copies", C.c_void_p), ("state", C.c_void_p),
    ]


class PageTensors(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
                ("bounds", C.c_void_p), ("bounds_scale", C.c_void_p)]


class CopyPagesParams(C.Structure):
    _fields_ = [
        ("n_copies", C.c_int), ("n_layers", C.c_int), ("kv_heads", C.c_int), ("head_dim", C.c_int), ("page_tokens", C.c_int), ("n_pages", C.c_int),
        ("page_stride", C.c_longlong), ("head_stride", C.c_longlong), ("token_stride", C.c_longlong), ("copies", C.c_void_p),
    ]


class ChooseParams(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("q_row", C.c_longlong), ("q_head", C.c_longlong), ("bounds", C.c_void_p), ("bounds_scale", C.c_void_p),
        ("chosen", C.c_void_p), ("chosen_row", C.c_longlong), ("chosen_head", C.c_longlong),
        ("count", C.c_int), ("first", C.c_int), ("last", C.c_int), ("reserved", C.c_int),
    ]


class ChosenPages(C.Structure):
    _fields_ = [("chosen", C.c_void_p), ("chosen_row", C.c_longlong), ("chosen_head", C.c_longlong), ("count", C.c_int), ("reserved", C.c_int)]


def packer(structure):
    """struct.Struct that writes all fields of a ctypes structure of ints, floats and addresses: a quarter of the time that filling in the
    structure takes (22 fields: 0.3 us against 1.3). An address that is missing is 0."""
    code = {C.c_int: "i", C.c_float: "f", C.c_longlong: "q", C.c_void_p: "P"}
    s = struct.Struct("".join(code[t] for _, t in structure._fields_))
    assert s.size == C.sizeof(structure)
    return s


# name -> (restype, argtypes); every symbol include/ogle_cuda.h declares
_vp = C.c_void_p
CUDA_SYMBOLS = {
    "ogle_cuda_status_string": (C.c_char_p, [C.c_int]),
    "ogle_cuda_set_wait_limit": (C.c_int, [C.c_long]),
    "ogle_cuda_last_contraction": (C.c_int, [C.POINTER(Contraction)]),
    "ogle_cuda_build_info": (C.c_char_p, []),
    "ogle_cuda_launch_count": (C.c_uint64, []),
    "ogle_cuda_last_error": (C.c_char_p, []),
    "ogle_cuda_conv2d_infer": (C.c_int, [C.POINTER(ConvParams)]),
    "ogle_cuda_conv2d_filter_bytes": (C.c_size_t, [C.POINTER(ConvParams)]),
    "ogle_cuda_conv2d_prepack": (C.c_int, [C.POINTER(ConvParams), _vp, _vp, _vp]),
    "ogle_cuda_conv2d": (C.c_int, [C.POINTER(ConvParams), _vp, _vp, _vp, _vp, _vp]),
    "ogle_cuda_conv2d_residual_supported": (C.c_int, [C.POINTER(ConvParams)]),
    "ogle_cuda_conv2d_residual": (C.c_int, [C.POINTER(ConvParams), _vp, _vp, _vp, _vp, C.c_int, _vp, _vp]),
    "ogle_cuda_conv2d_workspace_bytes": (C.c_size_t, [C.POINTER(ConvParams)]),
    "ogle_cuda_conv2d_ws": (C.c_int, [C.POINTER(ConvParams), _vp, _vp, _vp, _vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_conv2d_kernel_name": (C.c_char_p, [C.POINTER(ConvParams)]),
    "ogle_cuda_conv2d_pair_supported": (C.c_int, [C.POINTER(ConvParams)]),
    "ogle_cuda_conv2d_pair": (C.c_int, [C.POINTER(ConvParams), _vp, _vp, _vp, C.c_int, C.c_int, _vp, _vp, _vp]),
    "ogle_cuda_conv2d_pair_workspace_bytes": (C.c_size_t, [C.POINTER(ConvParams), C.c_int, C.c_int]),
    "ogle_cuda_conv2d_pair_ws": (C.c_int, [C.POINTER(ConvParams), _vp, _vp, _vp, C.c_int, C.c_int, _vp, _vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_pool_infer": (C.c_int, [C.POINTER(PoolParams)]),
    "ogle_cuda_pool": (C.c_int, [C.POINTER(PoolParams), _vp, _vp, _vp]),
    "ogle_cuda_batchnorm": (C.c_int, [_vp] * 6 + [C.c_long, C.c_int, C.c_int, C.c_float, _vp]),
    "ogle_cuda_relu": (C.c_int, [_vp, _vp, C.c_long, _vp]),
    "ogle_cuda_clip": (C.c_int, [_vp, _vp, C.c_long, C.c_float, C.c_float, _vp]),
    "ogle_cuda_add": (C.c_int, [_vp, _vp, _vp, C.c_long, _vp]),
    "ogle_cuda_add_act": (C.c_int, [_vp, _vp, _vp, C.c_long, C.c_int, C.c_float, C.c_float, _vp]),
    "ogle_cuda_gemm": (C.c_int, [C.POINTER(GemmParams), _vp, _vp, _vp, _vp, _vp]),
    "ogle_cuda_gemm_packed_b_bytes": (C.c_size_t, [C.POINTER(GemmParams)]),
    "ogle_cuda_gemm_pack_b": (C.c_int, [C.POINTER(GemmParams), _vp, _vp, _vp]),
    "ogle_cuda_gemm_packed": (C.c_int, [C.POINTER(GemmParams), _vp, _vp, _vp, _vp, _vp]),
    "ogle_cuda_gemm_ws": (C.c_int, [C.POINTER(GemmParams), _vp, _vp, _vp, _vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_gemm_static_max_bytes": (C.c_size_t, []),
    "ogle_cuda_gemm_static": (C.c_int, [C.POINTER(GemmParams), _vp, _vp, _vp, _vp, _vp]),
    "ogle_cuda_set_overlapped_launches": (C.c_int, [C.c_int]),
    "ogle_cuda_device_status": (C.c_int, []),
    "ogle_cuda_clear_device_status": (C.c_int, []),
    "ogle_cuda_device_status_detail": (C.c_int, []),
    "ogle_cuda_concat": (C.c_int, [C.POINTER(ConcatParams), C.POINTER(_vp), _vp, _vp]),
    "ogle_cuda_pad4": (C.c_int, [_vp, _vp, C.c_long, C.c_int, C.c_int, _vp]),
    "ogle_cuda_unpad4": (C.c_int, [_vp, _vp, C.c_long, C.c_int, C.c_int, _vp]),
    "ogle_cuda_preprocess_bgr8_batch": (C.c_int, [_vp, _vp, C.c_int, _vp, C.c_int, C.c_int, C.POINTER(C.c_float), _vp]),
    "ogle_cuda_preprocess_bgr8": (C.c_int, [_vp, C.c_int, C.c_int, C.c_int, _vp, C.c_int, C.c_int, C.POINTER(C.c_float), _vp]),
    "ogle_cuda_nchw_to_nhwc4": (C.c_int, [_vp, _vp] + [C.c_int] * 4 + [_vp]),
    "ogle_cuda_transpose": (C.c_int, [_vp, _vp, C.POINTER(C.c_int), C.POINTER(C.c_int), _vp]),
    "ogle_cuda_reshape": (C.c_int, [_vp, _vp, C.c_long, C.c_int, C.c_int, _vp]),
    "ogle_cuda_reshape_placed": (C.c_int, [_vp, _vp, C.c_long, C.c_int, C.c_int, C.c_long, C.c_long, _vp]),
    "ogle_cuda_ssd_decode": (C.c_int, [_vp, _vp, _vp, C.c_int, C.c_int, C.POINTER(C.c_float), _vp]),
    "ogle_cuda_ssd_detect": (C.c_int, [C.POINTER(DetectParams)] + [_vp] * 8),
    # the structures of these go as packed bytes (see packer) or by reference
    "ogle_cuda_kv_append": (C.c_int, [_vp, _vp, _vp]),
    "ogle_cuda_paged_attention_workspace_bytes": (C.c_size_t, [_vp, _vp]),
    "ogle_cuda_paged_attention": (C.c_int, [_vp, _vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_adjust_logits": (C.c_int, [_vp, _vp]),
    "ogle_cuda_beam_step_workspace_bytes": (C.c_size_t, [_vp]),
    "ogle_cuda_beam_step": (C.c_int, [_vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_advance_pages_workspace_bytes": (C.c_size_t, [_vp]),
    "ogle_cuda_advance_pages": (C.c_int, [_vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_compact_pages_workspace_bytes": (C.c_size_t, [_vp]),
    "ogle_cuda_compact_pages": (C.c_int, [_vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_copy_pages": (C.c_int, [_vp, _vp, _vp]),
    "ogle_cuda_page_bounds": (C.c_int, [_vp, _vp, _vp, _vp]),
    "ogle_cuda_choose_pages_workspace_bytes": (C.c_size_t, [_vp, _vp]),
    "ogle_cuda_choose_pages": (C.c_int, [_vp, _vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_sparse_attention_workspace_bytes": (C.c_size_t, [_vp, _vp, _vp]),
    "ogle_cuda_sparse_attention": (C.c_int, [_vp, _vp, _vp, _vp, C.c_size_t, _vp]),
    "ogle_cuda_ssd_decode_detect": (C.c_int, [C.POINTER(DetectParams), _vp, _vp, _vp, C.POINTER(C.c_float)] + [_vp] * 6),
}

_cuda = None


def cuda_lib():
    """Loads libogle_cuda.so (no GPU needed to load it) and types its symbols."""
    global _cuda
    if _cuda is None:
        if not os.path.exists(CUDA_LIB_PATH):
            raise RuntimeError(
                f"{CUDA_LIB_PATH} is missing: build it with `python -m ogle_b200.build` "
                "(nvcc, sm_100a). There is no fallback path.")
        lib = C.CDLL(CUDA_LIB_PATH, mode=C.RTLD_GLOBAL)
        for name, (res, args) in CUDA_SYMBOLS.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _cuda = lib
    return _cuda


class OgleError(RuntimeError):
    pass


def check(rc, what):
    if rc != 0:
        lib = cuda_lib()
        msg = lib.ogle_cuda_status_string(rc).decode()
        extra = lib.ogle_cuda_last_error().decode()
        raise OgleError(f"{what}: {msg} (status {rc}){' - ' + extra if extra and rc == -3 else ''}")
