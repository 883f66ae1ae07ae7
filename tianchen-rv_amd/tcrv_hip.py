"""ctypes binding of libtcrv_hip.so, the gfx950 runtime library.

The entry points keep the reference's emitted-kernel ABI (parameter roles and
order of ``tcrv_emitc_<kernel>_<variant>``, lib/Conversion/RVV/RVVToEmitC.cpp:
134-145, :258-268) and take caller-owned DEVICE pointers plus a HIP stream.
PyTorch is used only as the device-memory and stream allocator: tensors are
passed by ``data_ptr()``.

Loading fails loudly (``TcrvHipError``) when the library is missing: there is
no CPU fallback anywhere in this module.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional

HERE = os.path.dirname(os.path.abspath(__file__))
# TCRV_HIP_LIB selects another build of the library (same C-ABI).
LIB_PATH = os.environ.get("TCRV_HIP_LIB") or os.path.join(HERE, "libtcrv_hip.so")

QK = 32
Q8_0_BLOCK_BYTES = 34
Q4_0_BLOCK_BYTES = 18
Q4_0X16_BLOCK_BYTES = 288

OK = 0
ERR_NULL_POINTER = -1
ERR_BAD_SIZE = -2
ERR_MISALIGNED = -3
ERR_TOO_LARGE = -4
ERR_UNSUPPORTED = -5
ERR_SCRATCH_LIMIT = -6

# element types of the cache entries (TCRV_HIP_ELEM_*)
FLOAT_ELEM = {"f32": 7, "f16": 9, "bf16": 10}
ROPE_LAYOUT = {"interleaved": 0, "half": 1}
ROPE_SCALING = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
ACTIVATION = {"silu": 0, "gelu_tanh": 1, "gelu": 2, "relu": 3}

BINARY_ADD, BINARY_SUB, BINARY_MUL = 0, 1, 2
ELEM = {"i8": 0, "u8": 1, "i16": 2, "u16": 3, "i32": 4, "u32": 5, "i64": 6, "f32": 7, "f64": 8}


class TcrvHipError(RuntimeError):
    """A libtcrv_hip call returned a non-zero status, or the library is absent."""

    def __init__(self, status: int, message: str):
        super().__init__(message)
        self.status = status


_sz = ctypes.c_size_t
_p = ctypes.c_void_p
_i32 = ctypes.c_int32
_int = ctypes.c_int
_f32 = ctypes.c_float
_f64 = ctypes.c_double

# name -> argtypes (all return int status, except the string getters)
SIGNATURES = {
    "tcrv_hip_stream_synchronize": [_p],
    "tcrv_hip_add_f32": [_p, _p, _p, _sz, _p],
    "tcrv_hip_add_i32": [_p, _p, _p, _sz, _p],
    "tcrv_hip_binary": [_int, _int, _p, _p, _p, _sz, _p],
    "tcrv_hip_dequantize_row_q8_0": [_p, _p, _sz, _p],
    "tcrv_hip_dequantize_row_q4_0": [_p, _p, _sz, _p],
    "tcrv_hip_quantize_row_q8_0": [_sz, _p, _p, _p],
    "tcrv_hip_q8_0_q8_0_block_dot": [_sz, _p, _p, _p, _p],
    "tcrv_hip_q8_0_q8_0_block_dot_rows": [_sz, _p, _p, _sz, _p, _sz, _sz, _p],
    "tcrv_hip_q4_0_q8_0_block_dot": [_sz, _p, _sz, _p, _sz, _p, _sz, _i32, _p],
    "tcrv_hip_q4_0_q8_0_block_dot_rows": [_sz, _p, _p, _sz, _p, _sz, _sz, _p],
    "tcrv_hip_q8_0_q8_0_block_sums": [_sz, _p, _p, _sz, _p, _sz, _sz, _p],
    "tcrv_hip_q4_0_q8_0_block_sums": [_sz, _p, _p, _sz, _p, _sz, _sz, _p],
    "tcrv_hip_q4_0_q8_0_gemm": [_sz, _p, _p, _p, _sz, _sz, _sz, _sz, _sz, _p],
    "tcrv_hip_q4_0_q8_0_gemm_tile": [_sz, _p, _p, _p, _sz, _sz, _p],
    "tcrv_hip_gemv_q4_0_q8_0": [_sz, _p, _p, _sz, _p, _sz, _p],
    "tcrv_hip_gemv_q4_0_q8_0_shaped": [_sz, _p, _p, _sz, _p, _sz, _i32, _p],
    "tcrv_hip_q8_0_q8_0_gemm": [_sz, _p, _p, _p, _sz, _sz, _sz, _sz, _sz, _p],
    "tcrv_hip_pack_q4_0_to_q4_0x16": [_sz, _p, _p, _p],
    "tcrv_hip_pack_q8_0_to_q8_0x16": [_sz, _p, _p, _p],
    "tcrv_hip_repack_gemv_q4_0_q8_0": [_sz, _p, _p, _p, _sz, _p],
    "tcrv_hip_repack_gemv_q8_0_q8_0": [_sz, _p, _p, _p, _sz, _p],
    "tcrv_hip_repack_gemm_q4_0_q8_0": [_sz, _p, _p, _p, _sz, _sz, _sz, _p],
    "tcrv_hip_pack_q8_0_to_q8_0x4": [_sz, _sz, _p, _sz, _p, _p],
    "tcrv_hip_pack_q4_0_to_soa": [_sz, _sz, _p, _sz, _p, _p],
    "tcrv_hip_gemv_q4_0_soa_q8_0": [_sz, _p, _p, _p, _sz, _p],
    "tcrv_hip_packed_i4_offset_binary_x_i8_product_reduce": [_p, _p, _p, _p, _p, _sz, _p],
    "tcrv_hip_pack_q8_0_to_gemm_tiles": [_sz, _sz, _p, _sz, _p, _p],
    "tcrv_hip_q8_0_q8_0_gemm_tiles": [_sz, _p, _p, _p, _sz, _sz, _sz, _p],
    "tcrv_hip_q8_0_q8_0_gemm_ws": [_sz, _p, _p, _p, _sz, _sz, _sz, _sz, _sz, _p, _sz, _p],
    "tcrv_hip_q8_0_q8_0_gemm_noalloc": [_sz, _p, _p, _p, _sz, _sz, _sz, _sz, _sz, _p],
    "tcrv_hip_pack_q4_0_to_gemm_tiles": [_sz, _sz, _p, _sz, _p, _p],
    "tcrv_hip_q4_0_q8_0_gemm_tiles": [_sz, _p, _p, _p, _sz, _sz, _sz, _p],
    "tcrv_hip_q4_0_q8_0_gemm_ws": [_sz, _p, _p, _p, _sz, _sz, _sz, _sz, _sz, _p, _sz, _p],
    "tcrv_hip_rope_table": [_int, _sz, _f64, _f64, _f64, _f64, _f64, _f64, _p, _sz, _sz, _p, _p],
    "tcrv_hip_rope": [_int, _int, _p, _sz, _sz, _p, _sz, _sz, _p, _p, _sz, _sz, _sz, _sz, _sz,
                      _int, _p],
    "tcrv_hip_kv_tables": [_p, _p, _sz, _sz, _p, _sz, _p, _sz, _p, _p, _p, _p, _sz, _p, _p],
    "tcrv_hip_kv_store_q4_0": [_int, _p, _sz, _sz, _p, _sz, _sz, _int, _p, _p, _sz, _sz, _p, _p,
                               _sz, _sz, _sz, _sz, _sz, _p],
    "tcrv_hip_kv_load_q4_0": [_int, _p, _sz, _sz, _p, _p, _sz, _sz, _p, _sz, _sz, _sz, _sz, _sz,
                              _p],
    "tcrv_hip_attn_q4_0": [_int, _p, _sz, _sz, _p, _sz, _sz, _p, _sz, _p, _p, _sz, _sz, _sz, _sz,
                           _sz, _sz, _sz, _f32, _int, _sz, _p, _sz, _sz, _p, _sz, _p],
    "tcrv_hip_add_rms_norm": [_int, _p, _sz, _p, _sz, _p, _sz, _p, _f64, _p, _sz, _p, _sz, _sz,
                              _sz, _p],
    "tcrv_hip_gated_q4_0_q8_0": [_int, _int, _sz, _p, _sz, _p, _sz, _p, _p, _sz, _p, _sz, _sz, _sz,
                                 _p],
    "tcrv_hip_tree_tables": [_p, _p, _p, _sz, _p, _sz, _p, _sz, _p],
    "tcrv_hip_attn_tree_q4_0": [_int, _p, _sz, _sz, _p, _sz, _sz, _p, _sz, _p, _p, _p, _sz, _sz, _sz,
                                _sz, _sz, _sz, _sz, _sz, _f32, _sz, _p, _sz, _sz, _p, _sz, _p],
    "tcrv_hip_kv_keep_q4_0": [_p, _sz, _sz, _p, _sz, _p, _p, _p, _sz, _p, _sz, _sz, _sz, _sz, _p],
}
# size queries (return size_t)
SIZE_FUNCS = {"tcrv_hip_gemm_tiles_bytes": [_sz, _sz],
              "tcrv_hip_q8_0_q8_0_gemm_workspace_bytes": [_sz, _sz, _sz],
              "tcrv_hip_q4_0_q8_0_gemm_workspace_bytes": [_sz, _sz, _sz],
              "tcrv_hip_q8_0_q8_0_gemm_noalloc_max_bytes": [],
              "tcrv_hip_kv_q4_0_page_bytes": [_sz, _sz, _sz],
              "tcrv_hip_attn_q4_0_workspace_bytes": [_int, _sz, _sz, _sz, _sz, _sz, _sz, _sz],
              "tcrv_hip_attn_tree_q4_0_workspace_bytes": [_int, _sz, _sz, _sz, _sz, _sz, _sz,
                                                          _sz]}
STRING_FUNCS = {"tcrv_hip_status_string": [_int], "tcrv_hip_version": []}

_lib: Optional[ctypes.CDLL] = None
# symbol -> (foreign function, positions of its pointer arguments, argument
# count), of the library that _lib holds; filled by call().
_bound: dict = {}


def load(path: str = LIB_PATH) -> ctypes.CDLL:
    """Loads libtcrv_hip.so once; raises TcrvHipError if it is not built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise TcrvHipError(
            ERR_UNSUPPORTED,
            f"libtcrv_hip.so not found at {path}: run __graft_entry__.build() "
            "(make -C tianchen-rv_amd); there is no CPU fallback")
    # PyTorch-ROCm ships its own libamdhip64.  Importing torch first makes the
    # library bind to that same HIP runtime (one runtime per process, so torch's
    # streams and device pointers are valid here); loading the library first
    # maps the system runtime beside torch's, and the second runtime to
    # initialise finds no device.
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    lib = ctypes.CDLL(path)
    for name, argtypes in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = _int
    for name, argtypes in STRING_FUNCS.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = ctypes.c_char_p
    for name, argtypes in SIZE_FUNCS.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = _sz
    _bound.clear()
    _lib = lib
    return lib


def status_string(status: int) -> str:
    return load().tcrv_hip_status_string(status).decode()


def version() -> str:
    return load().tcrv_hip_version().decode()


def _check(name: str, status: int) -> int:
    if status != OK:
        raise TcrvHipError(status, f"{name} failed: {status} ({status_string(status)})")
    return status


def _ptr(t) -> int:
    """Device address of a torch tensor (or an int address / None)."""
    if t is None:
        return 0
    if isinstance(t, int):
        return t
    if not t.is_cuda:
        raise TcrvHipError(ERR_UNSUPPORTED, "libtcrv_hip takes device tensors only")
    return t.data_ptr()


def _raw_stream_getter():
    """() -> handle of torch's current stream on the current device.  torch's raw getters
    take 0.15 us; building the Stream object that torch.cuda.current_stream() returns takes
    2.7 us, as much as the launch itself."""
    import torch
    torch.cuda.current_stream()  # initialises the device, or raises
    try:
        device, raw = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    except AttributeError:
        return lambda: torch.cuda.current_stream().cuda_stream
    return lambda: raw(device())


_raw_stream = None


def _forget_raw_stream():
    """A forked child asks torch anew, which refuses a device that the parent initialised; the
    raw getters do not look."""
    global _raw_stream
    _raw_stream = None


if hasattr(os, "register_at_fork"):
    os.register_at_fork(after_in_child=_forget_raw_stream)


def _stream(stream) -> int:
    global _raw_stream
    if stream is None:
        if _raw_stream is None:
            _raw_stream = _raw_stream_getter()
        return _raw_stream()
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def _bind(name: str):
    fn = getattr(load(), name)
    argtypes = fn.argtypes
    bound = fn, tuple(i for i, t in enumerate(argtypes) if t is _p), len(argtypes)
    _bound[name] = bound
    return bound


def call(name: str, *args, check: bool = True) -> int:
    """Raw call by symbol name; tensor arguments are passed as device addresses.

    A 1024 x 1024 GEMV issued from Python: 7.7 -> 4.4 us a call, 3.2 of them the
    library's launch."""
    if _lib is None:
        load()
    fn, pointers, count = _bound.get(name) or _bind(name)
    conv = list(args[:count])
    for i in pointers:
        if i < len(conv):
            t = conv[i]
            if t.__class__ is not int:
                # a device tensor without _ptr's call: 0.1 us an argument
                conv[i] = t.data_ptr() if getattr(t, "is_cuda", False) else _ptr(t)
    status = fn(*conv)
    return _check(name, status) if check else status


# ---------------------------------------------------------------------------
# Typed wrappers in the reference's parameter order (plus a stream).
# ---------------------------------------------------------------------------

def add_f32(lhs, rhs, out, n: Optional[int] = None, stream=None):
    n = lhs.numel() if n is None else n
    return call("tcrv_hip_add_f32", lhs, rhs, out, n, _stream(stream))


def add_i32(lhs, rhs, out, n: Optional[int] = None, stream=None):
    n = lhs.numel() if n is None else n
    return call("tcrv_hip_add_i32", lhs, rhs, out, n, _stream(stream))


def binary(kind: int, elem: str, lhs, rhs, out, n: Optional[int] = None, stream=None):
    """tcrv_rvv.binary: kind BINARY_ADD/SUB/MUL, elem a key of ELEM."""
    n = lhs.numel() if n is None else n
    return call("tcrv_hip_binary", kind, ELEM[elem], lhs, rhs, out, n, _stream(stream))


def dequantize_row_q8_0(vx, y, n: int, stream=None):
    return call("tcrv_hip_dequantize_row_q8_0", vx, y, n, _stream(stream))


def dequantize_row_q4_0(vx, y, n: int, stream=None):
    return call("tcrv_hip_dequantize_row_q4_0", vx, y, n, _stream(stream))


def quantize_row_q8_0(n: int, x, vy, stream=None):
    return call("tcrv_hip_quantize_row_q8_0", n, x, vy, _stream(stream))


def packed_i4_offset_binary_x_i8_product_reduce(w, qlo, qhi, acc, out, n: int, stream=None):
    return call("tcrv_hip_packed_i4_offset_binary_x_i8_product_reduce", w, qlo, qhi, acc, out, n,
                _stream(stream))


def q8_0_q8_0_block_dot(n: int, s, vx, vy, stream=None):
    return call("tcrv_hip_q8_0_q8_0_block_dot", n, s, vx, vy, _stream(stream))


def q8_0_q8_0_block_dot_rows(n: int, s, vx, bx: int, vy, by: int, nrows: int, stream=None):
    return call("tcrv_hip_q8_0_q8_0_block_dot_rows", n, s, vx, bx, vy, by, nrows,
                _stream(stream))


def q4_0_q8_0_block_dot(n: int, s, bs: int, vx, bx: int, vy, by: int, nrc: int, stream=None):
    return call("tcrv_hip_q4_0_q8_0_block_dot", n, s, bs, vx, bx, vy, by, nrc,
                _stream(stream))


def q4_0_q8_0_block_dot_rows(n: int, s, vx, bx: int, vy, by: int, nrows: int, stream=None):
    return call("tcrv_hip_q4_0_q8_0_block_dot_rows", n, s, vx, bx, vy, by, nrows,
                _stream(stream))


def q8_0_q8_0_block_sums(n: int, sumi, vx, bx: int, vy, by: int, nrows: int, stream=None):
    return call("tcrv_hip_q8_0_q8_0_block_sums", n, sumi, vx, bx, vy, by, nrows,
                _stream(stream))


def q4_0_q8_0_block_sums(n: int, sumi, vx, bx: int, vy, by: int, nrows: int, stream=None):
    return call("tcrv_hip_q4_0_q8_0_block_sums", n, sumi, vx, bx, vy, by, nrows,
                _stream(stream))


def q4_0_q8_0_gemm(n: int, s, vx, vy, by: int, nr: int, nc: int, bx: int, bs: int,
                   stream=None):
    return call("tcrv_hip_q4_0_q8_0_gemm", n, s, vx, vy, by, nr, nc, bx, bs, _stream(stream))


def q4_0_q8_0_gemm_tile(n: int, s, vx, vy, by: int, m: int, stream=None):
    return call("tcrv_hip_q4_0_q8_0_gemm_tile", n, s, vx, vy, by, m, _stream(stream))


def gemv_q4_0_q8_0(n: int, s, vx, bx: int, vy, nr: int, stream=None):
    return call("tcrv_hip_gemv_q4_0_q8_0", n, s, vx, bx, vy, nr, _stream(stream))


def gemv_q4_0_q8_0_shaped(n: int, s, vx, bx: int, vy, nr: int, rows_per_wave: int, stream=None,
                          check: bool = True):
    return call("tcrv_hip_gemv_q4_0_q8_0_shaped", n, s, vx, bx, vy, nr, rows_per_wave,
                _stream(stream), check=check)


def q8_0_q8_0_gemm(n: int, s, vx, vy, by: int, nr: int, nc: int, bx: int, bs: int,
                   stream=None):
    return call("tcrv_hip_q8_0_q8_0_gemm", n, s, vx, vy, by, nr, nc, bx, bs, _stream(stream))


def pack_q4_0_to_q4_0x16(nblocks: int, src, dst, stream=None):
    return call("tcrv_hip_pack_q4_0_to_q4_0x16", nblocks, src, dst, _stream(stream))


def pack_q8_0_to_q8_0x16(nblocks: int, src, dst, stream=None):
    return call("tcrv_hip_pack_q8_0_to_q8_0x16", nblocks, src, dst, _stream(stream))


def repack_gemv_q4_0_q8_0(n: int, s, vx, vy, nc: int, stream=None):
    return call("tcrv_hip_repack_gemv_q4_0_q8_0", n, s, vx, vy, nc, _stream(stream))


def repack_gemv_q8_0_q8_0(n: int, s, vx, vy, nc: int, stream=None):
    return call("tcrv_hip_repack_gemv_q8_0_q8_0", n, s, vx, vy, nc, _stream(stream))


def repack_gemm_q4_0_q8_0(n: int, s, vx, vy, nr: int, nc: int, bs: int, stream=None):
    return call("tcrv_hip_repack_gemm_q4_0_q8_0", n, s, vx, vy, nr, nc, bs, _stream(stream))


def pack_q8_0_to_q8_0x4(nrows: int, nb: int, src, by: int, dst, stream=None):
    return call("tcrv_hip_pack_q8_0_to_q8_0x4", nrows, nb, src, by, dst, _stream(stream))


def pack_q4_0_to_soa(nrows: int, nb: int, src, bx: int, dst, stream=None):
    return call("tcrv_hip_pack_q4_0_to_soa", nrows, nb, src, bx, dst, _stream(stream))


def gemv_q4_0_soa_q8_0(n: int, s, vx, vy, nr: int, stream=None):
    return call("tcrv_hip_gemv_q4_0_soa_q8_0", n, s, vx, vy, nr, _stream(stream))


def gemm_tiles_bytes(nrows: int, nb: int) -> int:
    return load().tcrv_hip_gemm_tiles_bytes(nrows, nb)


def pack_q8_0_to_gemm_tiles(nrows: int, nb: int, src, bx: int, dst, stream=None):
    return call("tcrv_hip_pack_q8_0_to_gemm_tiles", nrows, nb, src, bx, dst, _stream(stream))


def q8_0_q8_0_gemm_tiles(n: int, s, tx, ty, nr: int, nc: int, bs: int, stream=None):
    return call("tcrv_hip_q8_0_q8_0_gemm_tiles", n, s, tx, ty, nr, nc, bs, _stream(stream))


def q8_0_q8_0_gemm_workspace_bytes(n: int, nr: int, nc: int) -> int:
    return load().tcrv_hip_q8_0_q8_0_gemm_workspace_bytes(n, nr, nc)


def q8_0_q8_0_gemm_ws(n: int, s, vx, vy, by: int, nr: int, nc: int, bx: int, bs: int, ws,
                      ws_bytes: int, stream=None):
    return call("tcrv_hip_q8_0_q8_0_gemm_ws", n, s, vx, vy, by, nr, nc, bx, bs, ws, ws_bytes,
                _stream(stream))


def q8_0_q8_0_gemm_noalloc_max_bytes() -> int:
    return load().tcrv_hip_q8_0_q8_0_gemm_noalloc_max_bytes()


def q8_0_q8_0_gemm_noalloc(n: int, s, vx, vy, by: int, nr: int, nc: int, bx: int, bs: int,
                           stream=None, check: bool = True):
    """tcrv_hip_q8_0_q8_0_gemm_ws with the library's fixed device scratch as the
    workspace (no allocation); returns the status when check is False."""
    return call("tcrv_hip_q8_0_q8_0_gemm_noalloc", n, s, vx, vy, by, nr, nc, bx, bs,
                _stream(stream), check=check)


def pack_q4_0_to_gemm_tiles(nrows: int, nb: int, src, bx: int, dst, stream=None):
    return call("tcrv_hip_pack_q4_0_to_gemm_tiles", nrows, nb, src, bx, dst, _stream(stream))


def q4_0_q8_0_gemm_tiles(n: int, s, tx, ty, nr: int, nc: int, bs: int, stream=None):
    return call("tcrv_hip_q4_0_q8_0_gemm_tiles", n, s, tx, ty, nr, nc, bs, _stream(stream))


def q4_0_q8_0_gemm_workspace_bytes(n: int, nr: int, nc: int) -> int:
    return load().tcrv_hip_q4_0_q8_0_gemm_workspace_bytes(n, nr, nc)


def q4_0_q8_0_gemm_ws(n: int, s, vx, vy, by: int, nr: int, nc: int, bx: int, bs: int, ws,
                      ws_bytes: int, stream=None):
    return call("tcrv_hip_q4_0_q8_0_gemm_ws", n, s, vx, vy, by, nr, nc, bx, bs, ws, ws_bytes,
                _stream(stream))


# ---- attention over a paged Q4_0 cache (include/tcrv_hip.h has the layouts).  elem is a key of
# FLOAT_ELEM, layout one of ROPE_LAYOUT; strides are in elements.

def kv_q4_0_page_bytes(page_size: int, kv_heads: int, head_dim: int) -> int:
    return load().tcrv_hip_kv_q4_0_page_bytes(page_size, kv_heads, head_dim)


def rope_table(n_dims: int, table, count: int, first: int = 0, base: float = 10000.0,
               scaling: str = "none", factor: float = 1.0, trained_context: float = 4096.0,
               beta_fast: float = 32.0, beta_slow: float = 1.0, amplitude: float = 0.0,
               divisors=None, stream=None):
    return call("tcrv_hip_rope_table", ROPE_SCALING[scaling], n_dims, base, factor,
                trained_context, beta_fast, beta_slow, amplitude, divisors, first, count, table,
                _stream(stream))


def rope(elem: str, layout: str, x, x_token: int, x_head: int, y, y_token: int, y_head: int,
         positions, table, table_rows: int, tokens: int, heads: int, head_dim: int, n_dims: int,
         inverse: bool = False, stream=None):
    return call("tcrv_hip_rope", FLOAT_ELEM[elem], ROPE_LAYOUT[layout], x, x_token, x_head, y,
                y_token, y_head, positions, table, table_rows, tokens, heads, head_dim, n_dims,
                inverse, _stream(stream))


def kv_tables(context, added, requests: int, page_size: int, free_pages, free_count: int,
              block_table, table_stride: int, first, length, positions, slots, max_tokens: int,
              taken, stream=None):
    return call("tcrv_hip_kv_tables", context, added, requests, page_size, free_pages, free_count,
                block_table, table_stride, first, length, positions, slots, max_tokens, taken,
                _stream(stream))


def kv_store_q4_0(elem: str, k, k_token: int, k_head: int, v, v_token: int, v_head: int,
                  layout: str, positions, table, table_rows: int, n_dims: int, slots, cache,
                  pages: int, page_size: int, tokens: int, kv_heads: int, head_dim: int,
                  stream=None):
    return call("tcrv_hip_kv_store_q4_0", FLOAT_ELEM[elem], k, k_token, k_head, v, v_token, v_head,
                ROPE_LAYOUT[layout], positions, table, table_rows, n_dims, slots, cache, pages,
                page_size, tokens, kv_heads, head_dim, _stream(stream))


def kv_load_q4_0(elem: str, cache, pages: int, page_size: int, slots, k, k_token: int, k_head: int,
                 v, v_token: int, v_head: int, tokens: int, kv_heads: int, head_dim: int,
                 stream=None):
    return call("tcrv_hip_kv_load_q4_0", FLOAT_ELEM[elem], cache, pages, page_size, slots, k,
                k_token, k_head, v, v_token, v_head, tokens, kv_heads, head_dim, _stream(stream))


def attn_q4_0_workspace_bytes(elem: str, requests: int, tokens: int, max_added: int,
                              max_length: int, heads: int, kv_heads: int, head_dim: int) -> int:
    return load().tcrv_hip_attn_q4_0_workspace_bytes(FLOAT_ELEM[elem], requests, tokens, max_added,
                                                     max_length, heads, kv_heads, head_dim)


def attn_q4_0(elem: str, q, q_token: int, q_head: int, cache, pages: int, page_size: int,
              block_table, table_stride: int, first, length, requests: int, tokens: int,
              max_added: int, max_length: int, heads: int, kv_heads: int, head_dim: int,
              scale: float, causal: bool, window: int, out, out_token: int, out_head: int, ws=None,
              ws_bytes: int = 0, stream=None):
    return call("tcrv_hip_attn_q4_0", FLOAT_ELEM[elem], q, q_token, q_head, cache, pages, page_size,
                block_table, table_stride, first, length, requests, tokens, max_added, max_length,
                heads, kv_heads, head_dim, scale, causal, window, out, out_token, out_head, ws,
                ws_bytes, _stream(stream))


# ---- between the quantized products of a step, and drafted tokens over the cache.  act is a key of
# ACTIVATION; None where an output is not wanted.

def add_rms_norm(elem: str, x, x_token: int, residual, residual_token: int, total, total_token: int,
                 weight, eps: float, y, y_token: int, q8, q8_token: int, tokens: int, n: int,
                 stream=None):
    return call("tcrv_hip_add_rms_norm", FLOAT_ELEM[elem], x, x_token, residual, residual_token, total,
                total_token, weight, eps, y, y_token, q8, q8_token, tokens, n, _stream(stream))


def gated_q4_0_q8_0(elem: str, act: str, n: int, out, out_token: int, q8, q8_token: int, gate, up,
                    bx: int, vy, by: int, nr: int, nc: int, stream=None):
    return call("tcrv_hip_gated_q4_0_q8_0", FLOAT_ELEM[elem], ACTIVATION[act], n, out, out_token, q8,
                q8_token, gate, up, bx, vy, by, nr, nc, _stream(stream))


def tree_tables(parents, first, length, requests: int, ancestors, words: int, positions,
                max_tokens: int, stream=None):
    return call("tcrv_hip_tree_tables", parents, first, length, requests, ancestors, words, positions,
                max_tokens, _stream(stream))


def attn_tree_q4_0_workspace_bytes(elem: str, requests: int, tokens: int, max_added: int,
                                   max_length: int, heads: int, kv_heads: int,
                                   head_dim: int) -> int:
    return load().tcrv_hip_attn_tree_q4_0_workspace_bytes(FLOAT_ELEM[elem], requests, tokens,
                                                          max_added, max_length, heads, kv_heads,
                                                          head_dim)


def attn_tree_q4_0(elem: str, q, q_token: int, q_head: int, cache, pages: int, page_size: int,
                   block_table, table_stride: int, first, length, ancestors, words: int,
                   requests: int, tokens: int, max_added: int, max_length: int, heads: int,
                   kv_heads: int, head_dim: int, scale: float, window: int, out, out_token: int,
                   out_head: int, ws=None, ws_bytes: int = 0, stream=None):
    return call("tcrv_hip_attn_tree_q4_0", FLOAT_ELEM[elem], q, q_token, q_head, cache, pages,
                page_size, block_table, table_stride, first, length, ancestors, words, requests,
                tokens, max_added, max_length, heads, kv_heads, head_dim, scale, window, out,
                out_token, out_head, ws, ws_bytes, _stream(stream))


def kv_keep_q4_0(cache, pages: int, page_size: int, block_table, table_stride: int, first, length,
                 path, path_stride: int, count, requests: int, max_added: int, kv_heads: int,
                 head_dim: int, stream=None):
    return call("tcrv_hip_kv_keep_q4_0", cache, pages, page_size, block_table, table_stride, first,
                length, path, path_stride, count, requests, max_added, kv_heads, head_dim,
                _stream(stream))


def synchronize(stream=None):
    return call("tcrv_hip_stream_synchronize", _stream(stream))


# ---------------------------------------------------------------------------
# libtcrv_hip_route.so: the host-side provider (include/tcrv_hip_route.h).
# ---------------------------------------------------------------------------
ROUTE_LIB_PATH = os.path.join(HERE, "libtcrv_hip_route.so")

QUANT = {"q4_0": 0, "q8_0": 1, "q4_K": 2}
M_DECODE, M_PREFILL = 0, 1
LAYOUT = {"plain": 0, "x16": 1}
ALGO = {0: "decline", 1: "decode_gemv", 2: "repack_gemv", 3: "mfma_gemm", 4: "repack_gemm"}

_cs = ctypes.c_char_p


class Schedule(ctypes.Structure):
    """tcrv_hip_schedule (include/tcrv_hip_route.h)."""
    _fields_ = [("op", _cs), ("m_regime", _int), ("kernel", _cs), ("knob", _cs),
                ("value", ctypes.c_int64), ("is_default", _int), ("entry", _cs),
                ("measured_us", ctypes.c_double), ("reason", _cs)]


ROUTE_SIGNATURES = {
    "tcrv_hip_route_select": ([_int, _int, _int, ctypes.POINTER(_int), ctypes.POINTER(_cs),
                               ctypes.POINTER(_cs)], _int),
    "tcrv_hip_route_m_regime": ([_sz], _int),
    "tcrv_hip_route_binary": ([_int, _int, ctypes.POINTER(_cs), ctypes.POINTER(_cs)], _int),
    "tcrv_hip_route_contraction": ([_int, _int, _sz, _p, _p, _p, _sz, _sz, _sz, _sz, _sz, _p,
                                    ctypes.POINTER(_int)], _int),
    "tcrv_hip_route_count": ([], _sz),
    "tcrv_hip_route_op": ([_sz], _cs),
    "tcrv_hip_route_entry": ([_sz], _cs),
    "tcrv_hip_route_param_count": ([_sz], _sz),
    "tcrv_hip_route_param": ([_sz, _sz, ctypes.POINTER(_cs), ctypes.POINTER(_cs),
                              ctypes.POINTER(_cs)], _int),
    "tcrv_hip_route_find": ([_cs], ctypes.c_long),
    "tcrv_hip_route_schedule_count": ([], _sz),
    "tcrv_hip_route_schedule": ([_sz, ctypes.POINTER(Schedule)], _int),
    "tcrv_hip_route_schedule_default": ([_cs, _int, _cs, ctypes.POINTER(ctypes.c_int64)], _int),
    "tcrv_hip_export_function": ([_cs, _cs, _cs, ctypes.POINTER(ctypes.c_int64), _sz, _int,
                                  ctypes.c_char_p, _sz, ctypes.POINTER(_sz)], _int),
    "tcrv_hip_export_prologue": ([], _cs),
}

EXPORT_DEFINITION, EXPORT_DECLARATION = 0, 1

_route: Optional[ctypes.CDLL] = None


def load_route(path: str = ROUTE_LIB_PATH) -> ctypes.CDLL:
    """Loads the route provider (after libtcrv_hip itself, so both share one
    HIP runtime); raises TcrvHipError if it is not built."""
    global _route
    if _route is not None:
        return _route
    load()
    if not os.path.exists(path):
        raise TcrvHipError(ERR_UNSUPPORTED, f"libtcrv_hip_route.so not found at {path}: run "
                           "__graft_entry__.build()")
    lib = ctypes.CDLL(path)
    for name, (argtypes, restype) in ROUTE_SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = restype
    _route = lib
    return lib


def route_select(quant: str, m_regime: int, layout: str):
    """(algorithm name, audit token, entry symbol or None) for typed facts."""
    lib = load_route()
    algo, reason, entry = _int(), _cs(), _cs()
    st = lib.tcrv_hip_route_select(QUANT[quant], m_regime, LAYOUT[layout], ctypes.byref(algo),
                                   ctypes.byref(reason), ctypes.byref(entry))
    _check("tcrv_hip_route_select", st)
    return ALGO[algo.value], reason.value.decode(), entry.value.decode() if entry.value else None


def route_binary(kind: int, elem: str):
    """(status, entry symbol or None, audit token) for tcrv_rvv.binary's typed
    facts: kind BINARY_ADD/SUB/MUL, elem a key of ELEM."""
    lib = load_route()
    entry, reason = _cs(), _cs()
    st = lib.tcrv_hip_route_binary(kind, ELEM[elem] if isinstance(elem, str) else elem,
                                   ctypes.byref(entry), ctypes.byref(reason))
    return st, entry.value.decode() if entry.value else None, reason.value.decode()


def route_table():
    """The op-identity route table: [{op, entry, params: [(c_name, c_type, role)]}]."""
    lib = load_route()
    rows = []
    for i in range(lib.tcrv_hip_route_count()):
        params = []
        for j in range(lib.tcrv_hip_route_param_count(i)):
            c_name, c_type, role = _cs(), _cs(), _cs()
            _check("tcrv_hip_route_param", lib.tcrv_hip_route_param(
                i, j, ctypes.byref(c_name), ctypes.byref(c_type), ctypes.byref(role)))
            params.append((c_name.value.decode(), c_type.value.decode(), role.value.decode()))
        rows.append({"op": lib.tcrv_hip_route_op(i).decode(),
                     "entry": lib.tcrv_hip_route_entry(i).decode(), "params": params})
    return rows


def route_schedules():
    """The schedule registry: one dict per (op, regime, knob, candidate value)."""
    lib = load_route()
    rows = []
    for i in range(lib.tcrv_hip_route_schedule_count()):
        r = Schedule()
        _check("tcrv_hip_route_schedule", lib.tcrv_hip_route_schedule(i, ctypes.byref(r)))
        rows.append({"op": r.op.decode(), "m_regime": r.m_regime, "kernel": r.kernel.decode(),
                     "knob": r.knob.decode(), "value": r.value, "is_default": bool(r.is_default),
                     "entry": r.entry.decode() if r.entry else None,
                     "measured_us": r.measured_us, "reason": r.reason.decode()})
    return rows


def route_schedule_default(op: str, m_regime: int, knob: str):
    """(status, the default value of `knob` for (op, m_regime) or None)."""
    v = ctypes.c_int64()
    st = load_route().tcrv_hip_route_schedule_default(op.encode(), m_regime, knob.encode(),
                                                      ctypes.byref(v))
    return st, (v.value if st == OK else None)


def export_function(op: str, kernel: str, variant: str, attrs=(), form: int = EXPORT_DEFINITION):
    """(status, C++ text) of the exported tcrv_emitc_<kernel>_<variant> for
    one selected variant of `op`; attrs are the baked-in op facts ({kind,
    element} for tcrv_rvv.binary, {activation_cols} for the GEMM tile)."""
    lib = load_route()
    arr = (ctypes.c_int64 * max(1, len(attrs)))(*attrs)
    need = _sz()
    st = lib.tcrv_hip_export_function(op.encode(), kernel.encode(), variant.encode(), arr,
                                      len(attrs), form, None, 0, ctypes.byref(need))
    if st != OK:
        return st, None
    buf = ctypes.create_string_buffer(need.value)
    st = lib.tcrv_hip_export_function(op.encode(), kernel.encode(), variant.encode(), arr,
                                      len(attrs), form, buf, need.value, None)
    return st, buf.value.decode()


def export_prologue() -> str:
    return load_route().tcrv_hip_export_prologue().decode()


def route_contraction(quant: str, layout: str, n: int, s, vx, vy, by: int, nr: int, nc: int,
                      bx: int, bs: int, stream=None, check: bool = True):
    """Runs a contraction (reference GEMM ABI) on the routed kernel; returns
    (status, algorithm name)."""
    lib = load_route()
    algo = _int(-1)
    st = lib.tcrv_hip_route_contraction(QUANT[quant], LAYOUT[layout], n, _ptr(s), _ptr(vx),
                                        _ptr(vy), by, nr, nc, bx, bs,
                                        _stream(stream) if stream != 0 else 0,
                                        ctypes.byref(algo))
    if check:
        _check("tcrv_hip_route_contraction", st)
    return st, ALGO.get(algo.value)
