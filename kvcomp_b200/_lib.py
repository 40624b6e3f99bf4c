"""ctypes binding of libkvcomp_b200.so (the C ABI declared in include/kvcomp_b200.h).

There is no fallback: if the library is missing or a call fails, an exception is raised.
"""
import ctypes as C
import os
import struct

from . import build as _build

KVC_OK = 0
FLAGS = {
    0x001: "ZERO_SCALE", 0x002: "MIN_OVERFLOW", 0x004: "CODE_OVERFLOW", 0x008: "SYMBOL_MISSING",
    0x010: "VECTOR_LONG", 0x020: "BLOCK_LONG", 0x040: "STREAM_FULL", 0x080: "BAD_STREAM",
    0x100: "CODE_TOO_LONG", 0x200: "NO_SYMBOLS", 0x400: "WAIT_TIMEOUT",
    0x800: "NO_PAGES", 0x1000: "BAD_PAGE", 0x2000: "BAD_LENGTH",
}
FLAG_ZERO_SCALE, FLAG_MIN_OVERFLOW, FLAG_CODE_OVERFLOW, FLAG_SYMBOL_MISSING = 0x1, 0x2, 0x4, 0x8
FLAG_VECTOR_LONG, FLAG_BLOCK_LONG, FLAG_STREAM_FULL, FLAG_BAD_STREAM = 0x10, 0x20, 0x40, 0x80
FLAG_CODE_TOO_LONG, FLAG_NO_SYMBOLS, FLAG_WAIT_TIMEOUT = 0x100, 0x200, 0x400
FLAG_NO_PAGES, FLAG_BAD_PAGE, FLAG_BAD_LENGTH = 0x800, 0x1000, 0x2000
# conditions under which the produced data cannot be trusted (the rest are informational)
FATAL_FLAGS = FLAG_CODE_OVERFLOW | FLAG_SYMBOL_MISSING | FLAG_BLOCK_LONG | FLAG_STREAM_FULL | \
    FLAG_BAD_STREAM | FLAG_CODE_TOO_LONG | FLAG_NO_SYMBOLS | FLAG_WAIT_TIMEOUT | FLAG_BAD_PAGE | FLAG_BAD_LENGTH

MODE_BLOCK, MODE_CHANNEL, MODE_TOKEN, MODE_VECTOR = 0, 1, 2, 3

LUT_BITS = 12
BOOK_OFF_ENC = 64
BOOK_OFF_REFTREE = BOOK_OFF_ENC + 2048
BOOK_OFF_TREE = BOOK_OFF_REFTREE + 1536
BOOK_OFF_LUT = BOOK_OFF_TREE + 2048
BOOK_BYTES = BOOK_OFF_LUT + 4 * (1 << LUT_BITS)


class QMeta(C.Structure):
    _fields_ = [("min_int", C.c_void_p), ("scale", C.c_void_p), ("min_bytes", C.c_int32),
                ("tok_div", C.c_int32), ("sj", C.c_int64), ("sb", C.c_int64), ("sh", C.c_int64),
                ("sc", C.c_int64)]


class Cache(C.Structure):
    _fields_ = [("encoded", C.c_void_p), ("encoded_bytes", C.c_int64), ("block_info", C.c_void_p),
                ("thread_info", C.c_void_p), ("book", C.c_void_p), ("q", QMeta),
                ("max_block_bytes", C.c_int32), ("reserved", C.c_int32)]


# the same layouts for the calls that a decode step makes (kvc_kv_store_packed, kvc_attn_decode_packed): packing all
# arguments at once costs a fifth of converting them one by one
CACHE_FIELDS = "7q2i4q2i"
KV_STORE_ARGS = struct.Struct("<11q")
ATTN_ARGS = struct.Struct("<" + 2 * CACHE_FIELDS + "12qfi")
STORE_ARGS = struct.Struct("<29q6ifi")
# (ops makes these calls through csrc/kvc_torch.cpp; for callers of the library by ctypes)
PAGE_PLAN_ARGS = struct.Struct("<18q")
PAGE_RELEASE_ARGS = struct.Struct("<14q")
ROTARY_ARGS = struct.Struct("<31q3if")
PAGED_ATTN_ARGS = struct.Struct("<29qfi")
SCALES = struct.Struct("<6q2i")
PAGE_SLOTS_ARGS = struct.Struct("<10q")
PAGE_SHIFT_ARGS = struct.Struct("<5q")
PREFIX_PLAN_ARGS = struct.Struct("<5q")
PAGED_ROWS_ARGS = struct.Struct("<2q6q2i19q2i")

ROTARY_HALF, ROTARY_INTERLEAVED = 0, 1
CODES_NONE, CODES_INT8, CODES_E4M3 = 0, 1, 2


class KvcError(RuntimeError):
    pass


_lib = None

_i64, _i32, _vp, _f32, _u32 = C.c_int64, C.c_int, C.c_void_p, C.c_float, C.c_uint32

_SIGNATURES = {
    "kvc_last_error": (C.c_char_p, []),
    "kvc_version": (_i32, []),
    "kvc_buffer_sizes": (_i32, [_i64, _i64, _i32, C.POINTER(_i64)]),
    "kvc_qmeta_make": (_i32, [_i32, _i32, _i64, _i64, _i64, _i64, _i64, C.POINTER(QMeta), C.POINTER(_i64)]),
    "kvc_quantize_workspace": (_i64, [_i32, _i32, _i64, _i64, _i64]),
    "kvc_quantize": (_i32, [_vp, _i64, _i64, _i64, _i64, _i32, _i32, _i64, _f32, _vp, _vp, _i32, _vp, _vp,
                            _vp, _i64, _vp, _vp]),
    "kvc_quant_minmax": (_i32, [_vp, _i64, _i64, _i64, _i64, _i32, _i32, _i64, _vp, _vp, _vp, _i64, _vp]),
    "kvc_quantize_ranged": (_i32, [_vp, _i64, _i64, _i64, _i64, _i32, _i32, _i64, _f32, _vp, _vp, _vp, _vp, _i32, _vp,
                                   _vp, _vp, _i64, _vp, _vp]),
    "kvc_rope_store": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _vp]),
    "kvc_rope_store_rows": (_i32, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i64, _vp]),
    "kvc_quantize_heads_fits": (_i32, [_i32, _i32, _i64, _i64, _i64, _i64, _i64]),
    "kvc_quantize_heads": (_i32, [_vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64, _i32, _i32, _i64, _f32, _vp, _vp, _i32, _vp, _vp, _vp, _vp]),
    "kvc_kv_store": (_i32, [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _vp]),
    "kvc_kv_store_packed": (_i32, [C.c_char_p, _vp]),
    "kvc_dequant": (_i32, [_vp, C.POINTER(QMeta), _i64, _i64, _i64, _i64, _vp, _vp]),
    "kvc_histogram": (_i32, [_vp, _i64, _vp, _vp]),
    "kvc_build_codebook": (_i32, [_vp, _vp, _vp]),
    "kvc_book_from_tree": (_i32, [_vp, _i64, _vp, _vp]),
    "kvc_encode_workspace": (_i64, [_i64, _i64, _i32]),
    "kvc_store_scratch": (_i64, [_i32, _i32, _i64, _i64, _i64, _i64, _i64, _i32]),
    "kvc_store_packed": (_i32, [C.c_char_p, _vp]),
    "kvc_stream_wait": (_i32, [_vp]),
    "kvc_encode_debug": (None, [_i32, _i32]),
    "kvc_encode": (_i32, [_vp, _i64, _i64, _i32, _vp, _i32, _u32, _vp, _vp, _vp, _i64, _vp, _vp, _i64, _vp, _vp]),
    "kvc_decode": (_i32, [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i32, _vp, _vp, _vp]),
    "kvc_decode_bounded": (_i32, [_vp, _i64, _vp, _vp, _vp, _i64, _i64, _i32, _u32, _vp, _vp, _vp]),
    "kvc_decode_values": (_i32, [C.POINTER(Cache), _i64, _i64, _i64, _i32, _vp, _vp, _vp]),
    "kvc_fused_qk": (_i32, [C.POINTER(Cache), _i64, _i64, _i64, _i64, _vp, _vp, _i32, _vp, _vp]),
    "kvc_fused_pv": (_i32, [C.POINTER(Cache), _i64, _i64, _i64, _i64, _vp, _vp, _vp, _vp]),
    "kvc_pv_sum": (_i32, [_vp, _i64, _i64, _i64, _vp, _vp]),
    "kvc_attn_workspace": (_i64, [_i64, _i64, _i32]),
    "kvc_attn_splits": (_i32, [_i64, _i64, _i64, _i32]),
    "kvc_attn_decode": (_i32, [C.POINTER(Cache), C.POINTER(Cache), _i64, _i64, _i64, _i64, _vp, _f32, _vp, _vp,
                               _i64, _vp, _i32, _vp, _i64, _vp, _vp]),
    "kvc_attn_decode_packed": (_i32, [C.c_char_p, _vp]),
    "kvc_attn_debug": (None, [_i32, _i32]),
    "kvc_decode_debug": (None, [_i32, _i32]),
    "kvc_attn_static_capacity": (_i64, []),
    "kvc_attn_decode_static": (_i32, [C.POINTER(Cache), C.POINTER(Cache), _i64, _i64, _i64, _i64, _vp, _f32, _vp, _vp,
                                      _i64, _vp, _i32, _vp, _vp]),
    "kvc_page_plan": (_i32, [C.c_char_p, _vp]),
    "kvc_page_release": (_i32, [C.c_char_p, _vp]),
    "kvc_rotary_store": (_i32, [C.c_char_p, _vp]),
    "kvc_paged_attn_cleared": (_i64, []),
    "kvc_paged_attn_workspace": (_i64, [_i64, _i64, _i64, _i64]),
    "kvc_paged_attn": (_i32, [C.c_char_p, _vp]),
    "kvc_paged_attn_rows": (_i32, [C.c_char_p, _vp, _i64, _vp]),
    "kvc_rotary_store_codes": (_i32, [C.c_char_p, C.c_char_p, _vp]),
    "kvc_page_slots": (_i32, [C.c_char_p, _vp]),
    "kvc_page_shift": (_i32, [C.c_char_p, _vp]),
    "kvc_paged_rows": (_i32, [C.c_char_p, _vp]),
    "kvc_paged_attn_codes": (_i32, [C.c_char_p, C.c_char_p, _vp, _i64, _vp]),
    "kvc_prefix_plan_words": (_i64, [_i64]),
    "kvc_prefix_plan": (_i32, [C.c_char_p, _vp]),
    "kvc_paged_attn_shared_workspace": (_i64, [_i64, _i64, _i64, _i64]),
    "kvc_paged_attn_shared": (_i32, [C.c_char_p, _vp, _vp, _i64, _vp]),
    "kvc_k_matvec": (_i32, [_vp, _vp, _vp, _i64, _i64, _vp]),
}

EXPORTS = tuple(_SIGNATURES)


def lib_path():
    return _build.LIB


def load():
    """Load (building first when the sources are newer) the CUDA library.  Raises if it cannot."""
    global _lib
    if _lib is not None:
        return _lib
    path = os.environ.get("KVCOMP_B200_LIB")          # an alternative build of the same library
    if not path:
        path = _build.LIB
        if _build.is_stale():
            path = _build.build(binding=False)
    if not os.path.exists(path):
        raise KvcError("libkvcomp_b200.so is missing and could not be built; there is no CPU fallback")
    lib = C.CDLL(path)
    for name, (res, args) in _SIGNATURES.items():
        fn = getattr(lib, name)      # AttributeError if the library does not export it
        fn.restype = res
        fn.argtypes = args
    _lib = lib
    return lib


_torch_calls = None


def torch_calls():
    """The paged cache's calls for torch (csrc/kvc_torch.cpp), built first when the source is newer, with this library's entries.  Raises if it cannot."""
    global _torch_calls
    if _torch_calls is not None:
        return _torch_calls
    import importlib.machinery
    import importlib.util

    import torch  # noqa: F401  (its libraries are loaded first)
    path = _build.build_binding()
    loader = importlib.machinery.ExtensionFileLoader("kvc_torch", path)
    module = importlib.util.module_from_spec(importlib.util.spec_from_file_location("kvc_torch", path, loader=loader))
    loader.exec_module(module)
    lib = load()
    module.init(KvcError, *(C.cast(getattr(lib, name), C.c_void_p).value
                            for name in ("kvc_page_plan", "kvc_page_release", "kvc_rotary_store", "kvc_paged_attn", "kvc_paged_attn_rows", "kvc_last_error",
                                         "kvc_rotary_store_codes", "kvc_page_slots", "kvc_page_shift", "kvc_paged_rows", "kvc_paged_attn_codes", "kvc_prefix_plan_words", "kvc_prefix_plan",
                                         "kvc_paged_attn_shared")))
    _torch_calls = module
    return module


def check(rc, what):
    if rc != KVC_OK:
        msg = load().kvc_last_error()
        raise KvcError("%s failed (code %d): %s" % (what, rc, msg.decode() if msg else ""))


def flag_names(status):
    return [n for bit, n in FLAGS.items() if status & bit]
