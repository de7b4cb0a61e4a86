"""ctypes binding of ``librpa_mi355x.so`` (declared in ``include/rpa_mi355x.h``).

There is no fallback: if the shared library is missing or does not load, importing the
op fails with an error that says how to build it.
"""

from __future__ import annotations

import ctypes
import os
import struct
from pathlib import Path

# RPA_LIBRARY points at another build of the same library (e.g. one compiled with different tile constants).
LIB_PATH = Path(os.environ.get("RPA_LIBRARY") or Path(__file__).resolve().parent / "lib" / "librpa_mi355x.so")

RPA_ABI_VERSION = 7
RPA_DTYPE_BF16, RPA_DTYPE_F32, RPA_DTYPE_FP8_E4M3, RPA_DTYPE_FP8_E5M2, RPA_DTYPE_INT8 = 0, 1, 2, 3, 4
RPA_COMPUTE_BF16, RPA_COMPUTE_F32 = 0, 1
RPA_FLAG_FORCE_GENERIC = 1
RPA_FLAG_FP32_LOGITS = 2
RPA_FLAG_PREFILL_TILES = 4
RPA_FLAG_PIPE_TILES = 8
RPA_FLAG_PLAIN_TILES = 16
RPA_FLAG_NO_LOGIT_STASH = 32

EXPORTED_SYMBOLS = (
    "rpa_abi_version",
    "rpa_last_error",
    "rpa_workspace_bytes",
    "rpa_kernel_path",
    "rpa_workspace_init",
    "rpa_fwd_launch",
    "rpa_fwd_launch_static",
    "rpa_static_scratch_bytes",
    "rpa_v3_launch",
    "rpa_v3_workspace_bytes",
    "rpa_page_attention_workspace_bytes",
    "rpa_page_attention_launch",
    "rpa_ragged_decode_workspace_bytes",
    "rpa_ragged_decode_launch",
    "rpa_quant_workspace_bytes",
    "rpa_quant_fwd_launch",
    "rpa_quant_update_launch",
    "rpa_quant_gather_launch",
    "rpa_block_tables_launch",
)


class RpaParams(ctypes.Structure):
    """Field-for-field image of ``struct RpaParams``."""

    _fields_ = [
        ("queries", ctypes.c_void_p),
        ("kv_pages", ctypes.c_void_p),
        ("context_lens", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("query_start_loc", ctypes.c_void_p),
        ("num_seqs", ctypes.c_void_p),
        ("sinks", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
        ("total_tokens", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("max_num_seqs", ctypes.c_int32),
        ("pages_per_seq", ctypes.c_int32),
        ("num_sinks", ctypes.c_int32),
        ("softmax_scale", ctypes.c_float),
        ("logits_soft_cap", ctypes.c_float),
        ("sliding_window", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("compute", ctypes.c_int32),
        ("num_queries_per_block", ctypes.c_int32),
        ("num_kv_pages_per_block", ctypes.c_int32),
        ("num_warps", ctypes.c_int32),
        ("num_stages", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
        ("q_scale", ctypes.c_float),
        ("k_scale", ctypes.c_float),
        ("v_scale", ctypes.c_float),
        ("kv_start", ctypes.c_void_p),
    ]


class RpaV3Params(ctypes.Structure):
    """Field-for-field image of ``struct RpaV3Params``."""

    _fields_ = [
        ("attn", RpaParams),
        ("new_keys", ctypes.c_void_p),
        ("new_values", ctypes.c_void_p),
        ("cache_dtype", ctypes.c_int32),
        ("cache_head_dim", ctypes.c_int32),
        ("cache_combined_heads", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


class RpaPageAttnParams(ctypes.Structure):
    """Field-for-field image of ``struct RpaPageAttnParams``."""

    _fields_ = [
        ("query", ctypes.c_void_p),
        ("key_cache", ctypes.c_void_p),
        ("value_cache", ctypes.c_void_p),
        ("context_lens", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
        ("num_seqs", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("block_size", ctypes.c_int32),
        ("num_blocks", ctypes.c_int32),
        ("max_blocks", ctypes.c_int32),
        ("attn_scale", ctypes.c_float),
        ("dtype", ctypes.c_int32),
        ("compute", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
    ]


class RpaRaggedDecodeParams(ctypes.Structure):
    """Field-for-field image of ``struct RpaRaggedDecodeParams``."""

    _fields_ = [
        ("query", ctypes.c_void_p),
        ("key", ctypes.c_void_p),
        ("value", ctypes.c_void_p),
        ("sequence_start", ctypes.c_void_p),
        ("sequence_end", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
        ("batch", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("seq_len", ctypes.c_int32),
        ("softmax_scale", ctypes.c_float),
        ("logits_soft_cap", ctypes.c_float),
        ("window_left", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("compute", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
        ("softmax_aux", ctypes.c_void_p),
        ("num_sinks", ctypes.c_int32),
        ("aux_rows", ctypes.c_int32),
    ]


class RpaQuantParams(ctypes.Structure):
    """Field-for-field image of ``struct RpaQuantParams``."""

    _fields_ = [
        ("queries", ctypes.c_void_p),
        ("kv_cache", ctypes.c_void_p),
        ("kv_scales", ctypes.c_void_p),
        ("context_lens", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("query_start_loc", ctypes.c_void_p),
        ("num_seqs", ctypes.c_void_p),
        ("sinks", ctypes.c_void_p),
        ("out", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_uint64),
        ("query_token_stride", ctypes.c_int64),
        ("query_head_stride", ctypes.c_int64),
        ("total_tokens", ctypes.c_int32),
        ("num_q_heads", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("scale_block", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("max_num_seqs", ctypes.c_int32),
        ("pages_per_seq", ctypes.c_int32),
        ("num_sinks", ctypes.c_int32),
        ("softmax_scale", ctypes.c_float),
        ("logits_soft_cap", ctypes.c_float),
        ("sliding_window", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("cache_dtype", ctypes.c_int32),
        ("flags", ctypes.c_uint32),
    ]


class RpaQuantUpdateParams(ctypes.Structure):
    """Field-for-field image of ``struct RpaQuantUpdateParams``."""

    _fields_ = [
        ("keys", ctypes.c_void_p),
        ("values", ctypes.c_void_p),
        ("kv_cache", ctypes.c_void_p),
        ("kv_scales", ctypes.c_void_p),
        ("slot_mapping", ctypes.c_void_p),
        ("key_token_stride", ctypes.c_int64),
        ("key_head_stride", ctypes.c_int64),
        ("value_token_stride", ctypes.c_int64),
        ("value_head_stride", ctypes.c_int64),
        ("total_tokens", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("scale_block", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("cache_dtype", ctypes.c_int32),
    ]


class RpaQuantGatherParams(ctypes.Structure):
    """Field-for-field image of ``struct RpaQuantGatherParams``."""

    _fields_ = [
        ("kv_cache", ctypes.c_void_p),
        ("kv_scales", ctypes.c_void_p),
        ("slot_mapping", ctypes.c_void_p),
        ("keys", ctypes.c_void_p),
        ("values", ctypes.c_void_p),
        ("total_tokens", ctypes.c_int32),
        ("num_kv_heads", ctypes.c_int32),
        ("head_dim", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("scale_block", ctypes.c_int32),
        ("num_pages", ctypes.c_int32),
        ("dtype", ctypes.c_int32),
        ("cache_dtype", ctypes.c_int32),
    ]


class RpaBlockTablesParams(ctypes.Structure):
    """Field-for-field image of ``struct RpaBlockTablesParams``."""

    _fields_ = [
        ("query_lens", ctypes.c_void_p),
        ("cached_lens", ctypes.c_void_p),
        ("block_tables", ctypes.c_void_p),
        ("free_pages", ctypes.c_void_p),
        ("free_state", ctypes.c_void_p),
        ("num_seqs", ctypes.c_void_p),
        ("query_start_loc", ctypes.c_void_p),
        ("context_lens", ctypes.c_void_p),
        ("slot_mapping", ctypes.c_void_p),
        ("positions", ctypes.c_void_p),
        ("admitted", ctypes.c_void_p),
        ("cached_lens_out", ctypes.c_void_p),
        ("free_state_out", ctypes.c_void_p),
        ("scratch", ctypes.c_void_p),
        ("max_num_seqs", ctypes.c_int32),
        ("pages_per_seq", ctypes.c_int32),
        ("num_free_slots", ctypes.c_int32),
        ("page_size", ctypes.c_int32),
        ("total_tokens", ctypes.c_int32),
        ("reserved", ctypes.c_int32),
    ]


RPA_MAX_SINK_KEYS = 64


class NativeLibraryError(RuntimeError):
    pass


_lib = None


def load() -> ctypes.CDLL:
    """Load the shared library once and declare the prototypes."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise NativeLibraryError(
            f"{LIB_PATH} is missing: build it with `python -m ejkernel_amd.build` "
            "(hipcc, --offload-arch=gfx950). There is no CPU or eager fallback."
        )
    try:
        lib = ctypes.CDLL(str(LIB_PATH))
    except OSError as e:  # pragma: no cover - depends on the host
        raise NativeLibraryError(f"cannot load {LIB_PATH}: {e}") from e
    for name in EXPORTED_SYMBOLS:
        if not hasattr(lib, name):
            raise NativeLibraryError(f"{LIB_PATH} does not export {name}")
    lib.rpa_abi_version.restype = ctypes.c_int
    lib.rpa_abi_version.argtypes = []
    lib.rpa_last_error.restype = ctypes.c_char_p
    lib.rpa_last_error.argtypes = []
    lib.rpa_workspace_bytes.restype = ctypes.c_uint64
    lib.rpa_workspace_bytes.argtypes = [ctypes.POINTER(RpaParams)]
    lib.rpa_kernel_path.restype = ctypes.c_int
    lib.rpa_kernel_path.argtypes = [ctypes.POINTER(RpaParams)]
    lib.rpa_workspace_init.restype = ctypes.c_int
    lib.rpa_workspace_init.argtypes = [ctypes.c_void_p, ctypes.c_uint64, ctypes.c_void_p]
    lib.rpa_fwd_launch.restype = ctypes.c_int
    lib.rpa_fwd_launch.argtypes = [ctypes.POINTER(RpaParams), ctypes.c_void_p]
    lib.rpa_fwd_launch_static.restype = ctypes.c_int
    lib.rpa_fwd_launch_static.argtypes = [ctypes.POINTER(RpaParams), ctypes.c_void_p]
    lib.rpa_static_scratch_bytes.restype = ctypes.c_uint64
    lib.rpa_static_scratch_bytes.argtypes = []
    lib.rpa_v3_workspace_bytes.restype = ctypes.c_uint64
    lib.rpa_v3_workspace_bytes.argtypes = [ctypes.POINTER(RpaV3Params)]
    lib.rpa_v3_launch.restype = ctypes.c_int
    lib.rpa_v3_launch.argtypes = [ctypes.POINTER(RpaV3Params), ctypes.c_void_p]
    lib.rpa_page_attention_workspace_bytes.restype = ctypes.c_uint64
    lib.rpa_page_attention_workspace_bytes.argtypes = [ctypes.POINTER(RpaPageAttnParams)]
    lib.rpa_page_attention_launch.restype = ctypes.c_int
    lib.rpa_page_attention_launch.argtypes = [ctypes.POINTER(RpaPageAttnParams), ctypes.c_void_p]
    lib.rpa_ragged_decode_workspace_bytes.restype = ctypes.c_uint64
    lib.rpa_ragged_decode_workspace_bytes.argtypes = [ctypes.POINTER(RpaRaggedDecodeParams)]
    lib.rpa_ragged_decode_launch.restype = ctypes.c_int
    lib.rpa_ragged_decode_launch.argtypes = [ctypes.POINTER(RpaRaggedDecodeParams), ctypes.c_void_p]
    lib.rpa_quant_workspace_bytes.restype = ctypes.c_uint64
    lib.rpa_quant_workspace_bytes.argtypes = [ctypes.POINTER(RpaQuantParams)]
    for name, params in (("rpa_quant_fwd_launch", RpaQuantParams), ("rpa_quant_update_launch", RpaQuantUpdateParams),
                         ("rpa_quant_gather_launch", RpaQuantGatherParams), ("rpa_block_tables_launch", RpaBlockTablesParams)):
        getattr(lib, name).restype = ctypes.c_int
        getattr(lib, name).argtypes = [ctypes.POINTER(params), ctypes.c_void_p]
    if lib.rpa_abi_version() != RPA_ABI_VERSION:
        raise NativeLibraryError(
            f"{LIB_PATH} has ABI version {lib.rpa_abi_version()}, this package expects {RPA_ABI_VERSION}: rebuild it"
        )
    _lib = lib
    return lib


_FORMATS = {ctypes.c_void_p: "Q", ctypes.c_uint64: "Q", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_uint32: "I", ctypes.c_float: "f"}


class Entry:
    """A C entry point of the shape ``int entry(const Params*, hipStream_t)``, called with the fields' values in order.

    The values are packed at once into the bytes of the struct, a fifth of what setting its fields one by one costs
    (pointers are integers here, 0 for null); a value outside its field's range is a ``ValueError``.
    """

    def __init__(self, name: str, params: type[ctypes.Structure]):
        self.name = name
        self.layout = struct.Struct("=" + "".join(_FORMATS[kind] for _, kind in params._fields_))
        assert self.layout.size == ctypes.sizeof(params), f"{params.__name__} has padding"
        self._function = None

    def __call__(self, stream: int, *values) -> None:
        fn = self._function
        if fn is None:
            fn = self._function = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)(ctypes.cast(getattr(load(), self.name), ctypes.c_void_p).value)
        try:
            packed = self.layout.pack(*values)
        except (struct.error, OverflowError) as e:
            raise ValueError(f"{self.name}: an argument is out of range: {e}") from None
        rc = fn(packed, stream)
        if rc != 0:
            kind = ValueError if rc in (-1, -2) else RuntimeError
            raise kind(f"{self.name} refused the call ({rc}): {last_error()}")


def last_error() -> str:
    return load().rpa_last_error().decode("utf-8", "replace")
