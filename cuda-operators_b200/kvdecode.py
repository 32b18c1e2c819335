"""Python host side of libkvdecode_b200.so (ctypes over the C ABI in include/kvdecode.h).

The reference (Murmurwkk/cuda-operators kv_cache/*.cu) is driven from host
C++ through ``extern "C"`` entry points; this module exposes the same entry
points with the same names and argument meaning (``solve``,
``kv_int8_split_launch``, ``kv_int8_simple_launch``) plus the extended API
(batched / GQA / ragged decode, quantise-on-append, row quantisation, LSE
combine). Device memory comes from torch tensors; torch is only plumbing
here -- every computation runs in the library's CUDA kernels. There is no
CPU fallback: if the shared library is missing, loading raises.
"""
from __future__ import annotations

import ctypes
import math
import os
import re
import subprocess
from pathlib import Path

HERE = Path(__file__).resolve().parent
ROOT = HERE.parent
LIB_PATH = HERE / "libkvdecode_b200.so"
HEADER = ROOT / "include" / "kvdecode.h"

KVD_FLAG_PARTIAL_OUT = 1
KVD_FLAG_Q_BF16 = 2
KVD_FLAG_Q_F16 = 4
KVD_FLAG_OUT_BF16 = 8
KVD_FLAG_OUT_F16 = 16
KVD_FLAG_QK_INT8 = 32
KVD_STATUS_OK = 0
KVD_STATUS_WAIT_TIMEOUT = 1
KVD_STATUS_CACHE_FULL = 2
KVD_STATUS_BAD_BLOCK = 4
KVD_STATUS_NO_BLOCKS = 8
CUDA_ERROR_INVALID_VALUE = 1

c_void_p = ctypes.c_void_p
c_int = ctypes.c_int
c_int32 = ctypes.c_int32
c_int64 = ctypes.c_int64
c_uint32 = ctypes.c_uint32
c_size_t = ctypes.c_size_t
c_float = ctypes.c_float


class DecodeDesc(ctypes.Structure):
    """Mirror of ``kvd_decode_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("num_q_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("max_seq_len", c_int32),
        ("flags", c_uint32),
        ("seq_lens", c_void_p),
        ("kv_stride_b", c_int64),
        ("kv_stride_h", c_int64),
        ("sc_stride_b", c_int64),
        ("sc_stride_h", c_int64),
        ("q_stride_b", c_int64),
        ("q_stride_h", c_int64),
        ("o_stride_b", c_int64),
        ("o_stride_h", c_int64),
        ("softmax_scale", c_float),
    ]


class AppendDesc(ctypes.Structure):
    """Mirror of ``kvd_append_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("capacity", c_int32),
        ("kv_stride_b", c_int64),
        ("kv_stride_h", c_int64),
        ("sc_stride_b", c_int64),
        ("sc_stride_h", c_int64),
        ("new_stride_b", c_int64),
        ("new_stride_h", c_int64),
    ]


class PagedDesc(ctypes.Structure):
    """Mirror of ``kvd_paged_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("num_q_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("block_size", c_int32),
        ("num_blocks", c_int32),
        ("max_blocks_per_seq", c_int32),
        ("flags", c_uint32),
        ("seq_lens", c_void_p),
        ("block_table", c_void_p),
        ("block_table_stride", c_int64),
        ("kv_stride_block", c_int64),
        ("kv_stride_h", c_int64),
        ("kv_stride_t", c_int64),
        ("sc_stride_block", c_int64),
        ("sc_stride_h", c_int64),
        ("q_stride_b", c_int64),
        ("q_stride_h", c_int64),
        ("o_stride_b", c_int64),
        ("o_stride_h", c_int64),
        ("softmax_scale", c_float),
    ]


class PrefillDesc(ctypes.Structure):
    """Mirror of ``kvd_prefill_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("num_q_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("max_seq_len", c_int32),
        ("max_queries", c_int32),
        ("flags", c_uint32),
        ("seq_lens", c_void_p),
        ("q_lens", c_void_p),
        ("kv_stride_b", c_int64),
        ("kv_stride_h", c_int64),
        ("sc_stride_b", c_int64),
        ("sc_stride_h", c_int64),
        ("q_stride_b", c_int64),
        ("q_stride_h", c_int64),
        ("q_stride_t", c_int64),
        ("o_stride_b", c_int64),
        ("o_stride_h", c_int64),
        ("o_stride_t", c_int64),
        ("softmax_scale", c_float),
    ]


class PagedPlanDesc(ctypes.Structure):
    """Mirror of ``kvd_paged_plan_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("block_size", c_int32),
        ("num_blocks", c_int32),
        ("max_blocks_per_seq", c_int32),
        ("num_slots", c_int32),
        ("block_table_stride", c_int64),
    ]


class PagedRowsDesc(ctypes.Structure):
    """Mirror of ``kvd_paged_rows_desc``."""

    _fields_ = [
        ("num_tokens", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("block_size", c_int32),
        ("num_blocks", c_int32),
        ("flags", c_uint32),
        ("row_stride_t", c_int64),
        ("row_stride_h", c_int64),
        ("kv_stride_block", c_int64),
        ("kv_stride_h", c_int64),
        ("kv_stride_t", c_int64),
        ("sc_stride_block", c_int64),
        ("sc_stride_h", c_int64),
    ]


class BlockSelectDesc(ctypes.Structure):
    """Mirror of ``kvd_block_select_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("num_q_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("block_size", c_int32),
        ("num_blocks", c_int32),
        ("max_blocks_per_seq", c_int32),
        ("budget", c_int32),
        ("first", c_int32),
        ("last", c_int32),
        ("flags", c_uint32),
        ("seq_lens", c_void_p),
        ("block_table", c_void_p),
        ("block_table_stride", c_int64),
        ("q_stride_b", c_int64),
        ("q_stride_h", c_int64),
    ]


class PagedPrefillDesc(ctypes.Structure):
    """Mirror of ``kvd_paged_prefill_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("num_q_heads", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("num_rows", c_int32),
        ("block_size", c_int32),
        ("num_blocks", c_int32),
        ("max_blocks_per_seq", c_int32),
        ("causal", c_int32),
        ("flags", c_uint32),
        ("seq_lens", c_void_p),
        ("row_starts", c_void_p),
        ("block_table", c_void_p),
        ("block_table_stride", c_int64),
        ("kv_stride_block", c_int64),
        ("kv_stride_h", c_int64),
        ("kv_stride_t", c_int64),
        ("sc_stride_block", c_int64),
        ("sc_stride_h", c_int64),
        ("q_stride_t", c_int64),
        ("q_stride_h", c_int64),
        ("o_stride_t", c_int64),
        ("o_stride_h", c_int64),
        ("softmax_scale", c_float),
    ]


class PagesDesc(ctypes.Structure):
    """Mirror of ``kvd_pages_desc``."""

    _fields_ = [
        ("batch", c_int32),
        ("num_kv_heads", c_int32),
        ("head_dim", c_int32),
        ("block_size", c_int32),
        ("num_blocks", c_int32),
        ("max_blocks_per_seq", c_int32),
        ("block_table_stride", c_int64),
        ("block_table_out_stride", c_int64),
        ("kv_stride_block", c_int64),
        ("kv_stride_h", c_int64),
        ("kv_stride_t", c_int64),
        ("sc_stride_block", c_int64),
        ("sc_stride_h", c_int64),
    ]


_SIGNATURES = {
    "solve": (None, [c_void_p] * 6 + [c_int] * 3),
    "kv_int8_split_launch": (c_int, [c_void_p] * 6 + [c_int] * 3 + [c_void_p, c_void_p]),
    "kv_int8_simple_launch": (c_int, [c_void_p] * 6 + [c_int] * 3 + [c_void_p, c_void_p]),
    "kvd_workspace_size": (c_size_t, [ctypes.POINTER(DecodeDesc)]),
    "kvd_decode_launch": (c_int, [ctypes.POINTER(DecodeDesc)] + [c_void_p] * 7 + [c_size_t, c_void_p]),
    "kvd_combine_launch": (c_int, [c_void_p, c_int, c_int64, c_int, c_int, c_void_p, c_int64, c_uint32, c_void_p]),
    "kvd_append_int8_launch": (c_int, [ctypes.POINTER(AppendDesc)] + [c_void_p] * 7 + [c_void_p]),
    "kvd_quantize_rows_launch": (c_int, [c_void_p, c_int64, c_int, c_int64, c_void_p, c_int64, c_void_p, c_void_p]),
    "kvd_device_status": (c_int, [ctypes.POINTER(c_int32)]),
    "kvd_last_launch_count": (c_int, []),
    "kvd_abi_version": (c_int, []),
    "kvd_error_string": (ctypes.c_char_p, [c_int]),
    "kvd_decode_launch_noalloc": (c_int, [ctypes.POINTER(DecodeDesc)] + [c_void_p] * 6 + [c_void_p]),
    "kvd_append_decode_launch": (c_int, [ctypes.POINTER(DecodeDesc), c_void_p, c_void_p, c_int64, c_int64]
                                 + [c_void_p] * 6 + [c_void_p, c_size_t, c_void_p]),
    "kvd_mgpu_get_unique_id": (c_int, [c_void_p]),
    "kvd_mgpu_comm_init": (c_int, [ctypes.POINTER(c_void_p), c_int, c_int, c_void_p]),
    "kvd_mgpu_comm_destroy": (c_int, [c_void_p]),
    "kvd_mgpu_seq_split_workspace_size": (c_size_t, [ctypes.POINTER(DecodeDesc), c_int]),
    "kvd_mgpu_seq_split_decode": (c_int, [ctypes.POINTER(DecodeDesc)] + [c_void_p] * 6
                                  + [c_void_p, c_size_t, c_void_p, c_int, c_void_p]),
    "kvd_mgpu_p2p_create": (c_int, [ctypes.POINTER(c_void_p), c_int, c_int, c_int, c_void_p, c_int, c_int]),
    "kvd_mgpu_p2p_destroy": (c_int, [c_void_p]),
    "kvd_mgpu_p2p_reset": (c_int, [c_void_p, c_void_p]),
    "kvd_mgpu_p2p_create_group": (c_int, [ctypes.POINTER(c_void_p), c_int, ctypes.POINTER(c_int), c_int, c_int, c_int]),
    "kvd_mgpu_p2p_workspace_size": (c_size_t, [ctypes.POINTER(DecodeDesc)]),
    "kvd_mgpu_p2p_seq_split_decode": (c_int, [c_void_p, ctypes.POINTER(DecodeDesc)] + [c_void_p] * 6
                                      + [c_void_p, c_size_t, c_void_p]),
    "kvd_prefill_workspace_size": (c_size_t, [ctypes.POINTER(PrefillDesc)]),
    "kvd_prefill_launch": (c_int, [ctypes.POINTER(PrefillDesc)] + [c_void_p] * 7 + [c_size_t, c_void_p]),
    "kvd_paged_workspace_size": (c_size_t, [ctypes.POINTER(PagedDesc)]),
    "kvd_paged_decode_launch": (c_int, [ctypes.POINTER(PagedDesc)] + [c_void_p] * 7 + [c_size_t, c_void_p]),
    "kvd_paged_append_int8_launch": (c_int, [ctypes.POINTER(PagedDesc), c_void_p, c_void_p, c_int64, c_int64]
                                     + [c_void_p] * 5 + [c_void_p]),
    "kvd_paged_plan_workspace_size": (c_size_t, [ctypes.POINTER(PagedPlanDesc)]),
    "kvd_paged_plan_launch": (c_int, [ctypes.POINTER(PagedPlanDesc)] + [c_void_p] * 10 + [c_size_t, c_void_p]),
    "kvd_paged_write_launch": (c_int, [ctypes.POINTER(PagedRowsDesc)] + [c_void_p] * 9 + [c_void_p]),
    "kvd_paged_read_launch": (c_int, [ctypes.POINTER(PagedRowsDesc)] + [c_void_p] * 7 + [c_void_p]),
    "kvd_block_select_workspace_size": (c_size_t, [ctypes.POINTER(BlockSelectDesc)]),
    "kvd_block_select_launch": (c_int, [ctypes.POINTER(BlockSelectDesc)] + [c_void_p] * 6 + [c_size_t, c_void_p]),
    "kvd_sparse_workspace_size": (c_size_t, [ctypes.POINTER(PagedDesc)]),
    "kvd_sparse_decode_launch": (c_int, [ctypes.POINTER(PagedDesc)] + [c_void_p] * 7 + [c_size_t, c_void_p]),
    "kvd_paged_prefill_workspace_size": (c_size_t, [ctypes.POINTER(PagedPrefillDesc)]),
    "kvd_paged_prefill_launch": (c_int, [ctypes.POINTER(PagedPrefillDesc)] + [c_void_p] * 7 + [c_size_t, c_void_p]),
    "kvd_paged_fork_workspace_size": (c_size_t, [ctypes.POINTER(PagesDesc)]),
    "kvd_paged_fork_launch": (c_int, [ctypes.POINTER(PagesDesc)] + [c_void_p] * 15 + [c_size_t, c_void_p]),
    "kvd_paged_compact_workspace_size": (c_size_t, [ctypes.POINTER(PagesDesc)]),
    "kvd_paged_compact_launch": (c_int, [ctypes.POINTER(PagesDesc)] + [c_void_p] * 14 + [c_size_t, c_void_p]),
}

NOALLOC_SCRATCH_BYTES = 512 * 1024

_lib = None


def build(force: bool = False) -> Path:
    """Compile libkvdecode_b200.so in place with nvcc (sm_100a)."""
    if force or not LIB_PATH.exists():
        subprocess.run(["make", "-C", str(HERE), "-j8"], check=True)
    return LIB_PATH


def lib() -> ctypes.CDLL:
    """Load the library (raises if it has not been built: there is no fallback)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is missing; build it with `make -C {HERE}`")
        handle = ctypes.CDLL(str(LIB_PATH))
        for name, (res, args) in _SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def header_functions() -> list[str]:
    """Names of every function declared in include/kvdecode.h."""
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    names = re.findall(r"^\s*(?:const\s+)?[A-Za-z_][\w\s\*]*?\b([A-Za-z_]\w*)\s*\([^;{]*\)\s*;", text, flags=re.M)
    return sorted(set(names))


class KvdError(RuntimeError):
    def __init__(self, code: int, where: str):
        self.code = code
        msg = lib().kvd_error_string(code)
        super().__init__(f"{where} failed: cuda error {code} ({msg.decode() if msg else '?'})")


def _check(code: int, where: str) -> None:
    if code != 0:
        raise KvdError(code, where)


def _ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


def _stream(stream) -> int | None:
    if stream is None:
        import torch

        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # a Stream object costs several microseconds
        return raw(torch.cuda.current_device()) if raw else torch.cuda.current_stream().cuda_stream
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


_torch = None


def _types():
    """(torch, int8, int32, int64, float32), looked up once: these calls are short, and so are their checks."""
    global _torch
    if _torch is None:
        import torch

        _torch = (torch, torch.int8, torch.int32, torch.int64, torch.float32)
    return _torch


_cuda = None


def _cuda_state():
    """(current stream's handle of a device, current device), looked up once: the public forms take longer."""
    global _cuda
    if _cuda is None:
        torch = _types()[0]
        _cuda = (getattr(torch._C, "_cuda_getCurrentRawStream", None)
                 or (lambda device: torch.cuda.current_stream(device).cuda_stream),
                 getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device)
    return _cuda


def _made(make, shape, dtype, t, stream, kept: bool = False):
    """A tensor of ``make`` (torch.empty, torch.zeros) on ``t``'s device for a call on ``stream``: made with that
    stream current, so that what fills it runs there too and its memory goes back to that stream's pool. ``kept``: the
    caller gets it, and may use it on the stream that is current now."""
    if stream is None or _stream(stream) == _cuda_state()[0](t.get_device()):
        return make(shape, dtype=dtype, device=t.device)
    cuda = _types()[0].cuda
    if not isinstance(stream, cuda.Stream):
        handle = _stream(stream)
        stream = cuda.ExternalStream(handle, t.device) if handle else cuda.default_stream(t.device)
    here = cuda.current_stream(t.device)
    with cuda.stream(stream):
        made = make(shape, dtype=dtype, device=t.device)
    if kept:
        made.record_stream(here)
    return made


def _out(shape, dtype, t, stream):
    """An output (``dtype``, default float32) of a call on ``stream`` whose data lie where ``t`` does."""
    types = _torch or _types()
    return _made(types[0].empty, shape, dtype or types[4], t, stream, True)


def _scratch(n: int, t, stream):
    """``n`` bytes (at least one) of scratch for a call on ``stream``."""
    torch = (_torch or _types())[0]
    return _made(torch.empty, n or 1, torch.uint8, t, stream)


# ---------------------------------------------------------------- reference ABI
def solve(Q, K_int8, V_int8, k_scale, v_scale, output, num_heads: int, seq_len: int, head_dim: int) -> None:
    """``solve`` of kv_cache/*.cu: default stream, no synchronisation, no return value."""
    lib().solve(_ptr(Q), _ptr(K_int8), _ptr(V_int8), _ptr(k_scale), _ptr(v_scale), _ptr(output),
                num_heads, seq_len, head_dim)


def kv_int8_split_launch(Q, K_int8, V_int8, k_scale, v_scale, output, num_heads, seq_len, head_dim, S,
                         stream=None) -> int:
    """Returns the cudaError_t code, like kv_cache/KV_int8_split_optimized.cu:268-292."""
    return lib().kv_int8_split_launch(_ptr(Q), _ptr(K_int8), _ptr(V_int8), _ptr(k_scale), _ptr(v_scale),
                                      _ptr(output), num_heads, seq_len, head_dim, _ptr(S), _stream(stream))


def kv_int8_simple_launch(Q, K_int8, V_int8, k_scale, v_scale, output, num_heads, seq_len, head_dim, S,
                          stream=None) -> int:
    """Returns the cudaError_t code, like kv_cache/new_kvint8.cu:85-100."""
    return lib().kv_int8_simple_launch(_ptr(Q), _ptr(K_int8), _ptr(V_int8), _ptr(k_scale), _ptr(v_scale),
                                       _ptr(output), num_heads, seq_len, head_dim, _ptr(S), _stream(stream))


# ----------------------------------------------------------------- extended API
def dtype_flags(q=None, out=None, partial: bool = False) -> int:
    """Decode flags for the element types of ``q`` and ``out`` (torch tensors:
    float32, bfloat16 or float16)."""
    import torch

    f = KVD_FLAG_PARTIAL_OUT if partial else 0
    if q is not None:
        if q.dtype not in _dtype_map():
            raise ValueError(f"unsupported query dtype {q.dtype}")
        f |= _dtype_map()[q.dtype]
    if out is not None and out.device.type != "meta":
        if out.dtype not in _dtype_map():
            raise ValueError(f"unsupported output dtype {out.dtype}")
        if partial and out.dtype != torch.float32:
            raise ValueError("partial records are float32")
        f |= _dtype_map()[out.dtype] << 2  # KVD_FLAG_OUT_* lie two bits above KVD_FLAG_Q_*
    return f


_dtypes = None


def _dtype_map() -> dict:
    """KVD_FLAG_Q_* of each element type."""
    global _dtypes
    if _dtypes is None:
        import torch

        _dtypes = {torch.float32: 0, torch.bfloat16: KVD_FLAG_Q_BF16, torch.float16: KVD_FLAG_Q_F16}
    return _dtypes


def make_desc(q, k, ks, out, seq_lens=None, max_seq_len: int | None = None, softmax_scale: float = 0.0,
              partial: bool = False, qk_int8: bool = False) -> DecodeDesc:
    """Descriptor for q [B,Hq,D], k/v [B,Hkv,cap,D] int8, ks/vs [B,Hkv,cap], out [B,Hq,D or D+4].
    ``qk_int8`` selects the INT8 Q.K mode (KVD_FLAG_QK_INT8: the query is rounded per head
    to int8 by the cache's quantiser rule)."""
    B, Hq, D = q.shape
    Bk, Hkv, cap, Dk = k.shape
    if Bk != B or Dk != D or Hq % Hkv:
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)}")
    if k.stride(3) != 1 or k.stride(2) != D or ks.stride(2) != 1 or q.stride(2) != 1 or out.stride(2) != 1:
        raise ValueError("token rows must be contiguous (d stride 1, K/V token stride D, scale token stride 1)")
    d = DecodeDesc()
    d.batch, d.num_q_heads, d.num_kv_heads, d.head_dim = B, Hq, Hkv, D
    d.max_seq_len = cap if max_seq_len is None else max_seq_len
    d.flags = dtype_flags(q, out, partial) | (KVD_FLAG_QK_INT8 if qk_int8 else 0)
    d.seq_lens = _ptr(seq_lens)
    d.kv_stride_b, d.kv_stride_h = k.stride(0), k.stride(1)
    d.sc_stride_b, d.sc_stride_h = ks.stride(0), ks.stride(1)
    d.q_stride_b, d.q_stride_h = q.stride(0), q.stride(1)
    d.o_stride_b, d.o_stride_h = out.stride(0), out.stride(1)
    d.softmax_scale = softmax_scale
    return d


def workspace_size(desc: DecodeDesc) -> int:
    return int(lib().kvd_workspace_size(ctypes.byref(desc)))


def decode(q, k, v, ks, vs, out=None, seq_lens=None, softmax_scale: float = 0.0, partial: bool = False,
           workspace=None, max_seq_len: int | None = None, stream=None, out_dtype=None, qk_int8: bool = False):
    """Split-KV INT8 decode attention; returns ``out`` ([B,Hq,D], or [B,Hq,D+4] records if partial).
    ``q`` may be float32, bfloat16 or float16; the output type is ``out``'s (or ``out_dtype``,
    default float32). ``qk_int8`` selects the INT8 Q.K mode (looser, stated tolerance)."""
    B, Hq, D = q.shape
    if out is None:
        out = _out((B, Hq, D + 4 if partial else D), out_dtype, q, stream)
    if v.stride() != k.stride() or vs.stride() != ks.stride():
        raise ValueError("K/V and k_scale/v_scale must share strides")
    desc = make_desc(q, k, ks, out, seq_lens, max_seq_len, softmax_scale, partial, qk_int8)
    if workspace is None:
        n = workspace_size(desc)
        workspace = _scratch(n, q, stream)
    rc = lib().kvd_decode_launch(ctypes.byref(desc), _ptr(q), _ptr(k), _ptr(v), _ptr(ks), _ptr(vs), _ptr(out),
                                 _ptr(workspace), workspace.numel(), _stream(stream))
    _check(rc, "kvd_decode_launch")
    return out


def decode_noalloc(q, k, v, ks, vs, out, seq_lens=None, softmax_scale: float = 0.0, partial: bool = False,
                   max_seq_len: int | None = None, stream=None):
    """Same decode for callers that may not allocate device memory: the
    library's fixed scratch array replaces the workspace, so this allocates
    nothing (``out`` must be given). Calls that overlap on the GPU race on that
    array; the first call on a device should not be inside a stream capture."""
    if v.stride() != k.stride() or vs.stride() != ks.stride():
        raise ValueError("K/V and k_scale/v_scale must share strides")
    desc = make_desc(q, k, ks, out, seq_lens, max_seq_len, softmax_scale, partial)
    rc = lib().kvd_decode_launch_noalloc(ctypes.byref(desc), _ptr(q), _ptr(k), _ptr(v), _ptr(ks), _ptr(vs),
                                         _ptr(out), _stream(stream))
    _check(rc, "kvd_decode_launch_noalloc")
    return out


def combine(parts, out=None, partial: bool = False, stream=None, out_dtype=None):
    """LSE-combine records ``parts`` [P, H, D+4] into out [H, D] (or [H, D+4] records)."""
    P, H, R = parts.shape
    D = R - 4
    if out is None:
        out = _out((H, R if partial else D), out_dtype, parts, stream)
    rc = lib().kvd_combine_launch(_ptr(parts), P, parts.stride(0), H, D, _ptr(out), out.stride(0),
                                  dtype_flags(None, out, partial), _stream(stream))
    _check(rc, "kvd_combine_launch")
    return out


def append(k_new, v_new, K, V, ks, vs, seq_lens, stream=None) -> None:
    """Quantise-on-append of one token per (b, h): k_new/v_new [B,Hkv,D] fp32 into the cache."""
    B, H, D = k_new.shape
    d = AppendDesc()
    d.batch, d.num_kv_heads, d.head_dim, d.capacity = B, H, D, K.shape[2]
    d.kv_stride_b, d.kv_stride_h = K.stride(0), K.stride(1)
    d.sc_stride_b, d.sc_stride_h = ks.stride(0), ks.stride(1)
    d.new_stride_b, d.new_stride_h = k_new.stride(0), k_new.stride(1)
    if v_new.stride() != k_new.stride() or V.stride() != K.stride() or vs.stride() != ks.stride():
        raise ValueError("K/V (and their scales, and the new rows) must share strides")
    rc = lib().kvd_append_int8_launch(ctypes.byref(d), _ptr(k_new), _ptr(v_new), _ptr(K), _ptr(V), _ptr(ks),
                                      _ptr(vs), _ptr(seq_lens), _stream(stream))
    _check(rc, "kvd_append_int8_launch")


def append_decode(k_new, v_new, q, k, v, ks, vs, seq_lens, out=None, workspace=None, softmax_scale: float = 0.0,
                  partial: bool = False, stream=None, out_dtype=None, qk_int8: bool = False):
    """Quantise-on-append of one token per (b, kv head) and the decode over the grown
    cache in one decode launch (``kvd_append_decode_launch``); ``seq_lens`` is updated."""
    B, Hq, D = q.shape
    if out is None:
        out = _out((B, Hq, D + 4 if partial else D), out_dtype, q, stream)
    if v.stride() != k.stride() or vs.stride() != ks.stride() or v_new.stride() != k_new.stride():
        raise ValueError("K/V (and their scales, and the new rows) must share strides")
    desc = make_desc(q, k, ks, out, seq_lens, None, softmax_scale, partial, qk_int8)
    if workspace is None:
        workspace = _scratch(workspace_size(desc), q, stream)
    rc = lib().kvd_append_decode_launch(ctypes.byref(desc), _ptr(k_new), _ptr(v_new), k_new.stride(0),
                                        k_new.stride(1), _ptr(q), _ptr(k), _ptr(v), _ptr(ks), _ptr(vs), _ptr(out),
                                        _ptr(workspace), workspace.numel(), _stream(stream))
    _check(rc, "kvd_append_decode_launch")
    return out


def make_prefill_desc(q, k, ks, out, seq_lens=None, q_lens=None, softmax_scale: float = 0.0) -> PrefillDesc:
    """Descriptor for q [B,Hq,Lq,D], k/v [B,Hkv,cap,D] int8, ks/vs [B,Hkv,cap], out [B,Hq,Lq,D]."""
    B, Hq, Lq, D = q.shape
    Bk, Hkv, cap, Dk = k.shape
    if Bk != B or Dk != D or Hq % Hkv or tuple(out.shape) != (B, Hq, Lq, D):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k{tuple(k.shape)} out{tuple(out.shape)}")
    if k.stride(3) != 1 or k.stride(2) != D or ks.stride(2) != 1 or q.stride(3) != 1 or out.stride(3) != 1:
        raise ValueError("token rows must be contiguous")
    d = PrefillDesc()
    d.batch, d.num_q_heads, d.num_kv_heads, d.head_dim = B, Hq, Hkv, D
    d.max_seq_len, d.max_queries = cap, Lq
    d.flags = dtype_flags(q, out)
    d.seq_lens, d.q_lens = _ptr(seq_lens), _ptr(q_lens)
    d.kv_stride_b, d.kv_stride_h = k.stride(0), k.stride(1)
    d.sc_stride_b, d.sc_stride_h = ks.stride(0), ks.stride(1)
    d.q_stride_b, d.q_stride_h, d.q_stride_t = q.stride(0), q.stride(1), q.stride(2)
    d.o_stride_b, d.o_stride_h, d.o_stride_t = out.stride(0), out.stride(1), out.stride(2)
    d.softmax_scale = softmax_scale
    return d


def prefill(q, k, v, ks, vs, seq_lens=None, q_lens=None, out=None, softmax_scale: float = 0.0, out_dtype=None,
            workspace=None, stream=None):
    """Causal prefill attention over the INT8 cache; q [B,Hq,Lq,D] holds the last q_lens[b]
    (default Lq) of the seq_lens[b] (default cap) cached tokens. Returns out [B,Hq,Lq,D]."""
    if out is None:
        out = _out(q.shape, out_dtype, q, stream)
    if v.stride() != k.stride() or vs.stride() != ks.stride():
        raise ValueError("K/V and k_scale/v_scale must share strides")
    desc = make_prefill_desc(q, k, ks, out, seq_lens, q_lens, softmax_scale)
    if workspace is None:
        workspace = _scratch(int(lib().kvd_prefill_workspace_size(ctypes.byref(desc))), q, stream)
    rc = lib().kvd_prefill_launch(ctypes.byref(desc), _ptr(q), _ptr(k), _ptr(v), _ptr(ks), _ptr(vs), _ptr(out),
                                  _ptr(workspace), workspace.numel(), _stream(stream))
    _check(rc, "kvd_prefill_launch")
    return out


def quantize_rows(x, codes=None, scales=None, stream=None):
    """Quantise a 2-D fp32 tensor row by row; returns (codes int8 like x, scales [rows])."""
    import torch

    rows, dim = x.shape
    if codes is None:
        codes = _out((rows, dim), torch.int8, x, stream)
    if scales is None:
        scales = _out((rows,), torch.float32, x, stream)
    rc = lib().kvd_quantize_rows_launch(_ptr(x), rows, dim, x.stride(0), _ptr(codes), codes.stride(0),
                                        _ptr(scales), _stream(stream))
    _check(rc, "kvd_quantize_rows_launch")
    return codes, scales


# ------------------------------------------------------------------ paged cache
def make_paged_desc(q, k_pool, ks_pool, out, block_table, seq_lens, layout: str = "bhtd",
                    softmax_scale: float = 0.0, partial: bool = False, qk_int8: bool = False) -> PagedDesc:
    """Descriptor for a paged cache. ``k_pool`` is [blocks, Hkv, block_size, D]
    (layout "bhtd") or [blocks, block_size, Hkv, D] (layout "bthd"); scale pools
    are [blocks, Hkv, block_size]; ``block_table`` is int32 [B, max_blocks]."""
    B, Hq, D = q.shape
    if layout == "bhtd":
        NB, Hkv, bs, Dk = k_pool.shape
        s_blk, s_h, s_t = k_pool.stride(0), k_pool.stride(1), k_pool.stride(2)
    elif layout == "bthd":
        NB, bs, Hkv, Dk = k_pool.shape
        s_blk, s_t, s_h = k_pool.stride(0), k_pool.stride(1), k_pool.stride(2)
    else:
        raise ValueError(f"unknown pool layout {layout!r}")
    if Dk != D or Hq % Hkv or tuple(ks_pool.shape) != (NB, Hkv, bs):
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k_pool{tuple(k_pool.shape)} ks{tuple(ks_pool.shape)}")
    if k_pool.stride(3) != 1 or ks_pool.stride(2) != 1 or q.stride(2) != 1 or out.stride(2) != 1:
        raise ValueError("dims and scale tokens must be contiguous")
    if block_table.dim() != 2 or block_table.shape[0] != B or block_table.stride(1) != 1:
        raise ValueError("block_table must be int32 [B, max_blocks] with contiguous rows")
    d = PagedDesc()
    d.batch, d.num_q_heads, d.num_kv_heads, d.head_dim = B, Hq, Hkv, D
    d.block_size, d.num_blocks, d.max_blocks_per_seq = bs, NB, block_table.shape[1]
    d.flags = dtype_flags(q if q.device.type != "meta" else None, out, partial) | (KVD_FLAG_QK_INT8 if qk_int8 else 0)
    d.seq_lens, d.block_table = _ptr(seq_lens), _ptr(block_table)
    d.block_table_stride = block_table.stride(0)
    d.kv_stride_block, d.kv_stride_h, d.kv_stride_t = s_blk, s_h, s_t
    d.sc_stride_block, d.sc_stride_h = ks_pool.stride(0), ks_pool.stride(1)
    d.q_stride_b, d.q_stride_h = q.stride(0), q.stride(1)
    d.o_stride_b, d.o_stride_h = out.stride(0), out.stride(1)
    d.softmax_scale = softmax_scale
    return d


def paged_workspace_size(desc: PagedDesc) -> int:
    return int(lib().kvd_paged_workspace_size(ctypes.byref(desc)))


def paged_decode(q, k_pool, v_pool, ks_pool, vs_pool, block_table, seq_lens, out=None, layout: str = "bhtd",
                 softmax_scale: float = 0.0, partial: bool = False, workspace=None, stream=None, out_dtype=None,
                 qk_int8: bool = False):
    """INT8 decode attention over a paged cache; returns ``out`` [B,Hq,D] (or records)."""
    B, Hq, D = q.shape
    if out is None:
        out = _out((B, Hq, D + 4 if partial else D), out_dtype, q, stream)
    if v_pool.stride() != k_pool.stride() or vs_pool.stride() != ks_pool.stride():
        raise ValueError("K/V pools and their scale pools must share strides")
    desc = make_paged_desc(q, k_pool, ks_pool, out, block_table, seq_lens, layout, softmax_scale, partial, qk_int8)
    if workspace is None:
        workspace = _scratch(paged_workspace_size(desc), q, stream)
    rc = lib().kvd_paged_decode_launch(ctypes.byref(desc), _ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(ks_pool),
                                       _ptr(vs_pool), _ptr(out), _ptr(workspace), workspace.numel(),
                                       _stream(stream))
    _check(rc, "kvd_paged_decode_launch")
    return out


def paged_append(k_new, v_new, k_pool, v_pool, ks_pool, vs_pool, block_table, seq_lens, layout: str = "bhtd",
                 stream=None) -> None:
    """Quantise-on-append of one token per (b, kv head) into a paged cache."""
    import torch

    B, Hkv, D = k_new.shape
    if v_new.stride() != k_new.stride() or v_pool.stride() != k_pool.stride() or vs_pool.stride() != ks_pool.stride():
        raise ValueError("K/V (and their scales, and the new rows) must share strides")
    q_like = torch.empty((B, Hkv, D), dtype=torch.float32, device="meta")
    desc = make_paged_desc(q_like, k_pool, ks_pool, q_like, block_table, seq_lens, layout)
    rc = lib().kvd_paged_append_int8_launch(ctypes.byref(desc), _ptr(k_new), _ptr(v_new), k_new.stride(0),
                                            k_new.stride(1), _ptr(k_pool), _ptr(v_pool), _ptr(ks_pool),
                                            _ptr(vs_pool), _ptr(seq_lens), _stream(stream))
    _check(rc, "kvd_paged_append_int8_launch")


# ------------------------------------------- paged serving steps on the GPU
def _row_flags(dtype) -> int:
    """KVD_FLAG_Q_* of a row type."""
    f = _dtype_map().get(dtype)
    if f is None:
        raise ValueError(f"unsupported row dtype {dtype}")
    return f


def _want(device: int, dtype, *wanted) -> None:
    """Contiguous tensors of this device and type: a (tensor, shape, name) each, tensors that are None aside."""
    for t, shape, what in wanted:
        if t is None:
            continue
        if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
            raise ValueError(f"{what} must be contiguous {dtype} of shape {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
        if t.get_device() != device:
            raise _elsewhere(t)


def _own_scratch(device: int, workspace) -> None:
    """A caller's workspace: bytes that lie together, on the device."""
    if workspace is None:
        return
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    if workspace.get_device() != device:
        raise _elsewhere(workspace)


def _elsewhere(t) -> ValueError:
    return ValueError(f"all tensors must be on one device, got another on {t.device}")


def _handle(device: int, stream) -> int:
    """The given stream, or the current one, of the tensors' device, which has to be the current device: launches go
    there, and their sizes are its own."""
    raw_stream, current_device = _cuda or _cuda_state()
    if device < 0 or current_device() != device:
        raise ValueError("tensors must be on the current CUDA device")
    return raw_stream(device) if stream is None else _stream(stream)


def _pools(device: int, k_pool, v_pool, ks_pool, vs_pool, layout: str):
    """(blocks, heads, block_size, head_dim, block stride, head stride, token stride, scale strides) of K and V pools."""
    _, i8, _, _, f32 = _torch or _types()
    shape, strides, sc_shape, sc_strides = k_pool.shape, k_pool.stride(), ks_pool.shape, ks_pool.stride()
    if layout == "bhtd":
        NB, H, bs, D = shape
        s_blk, s_h, s_t, s_d = strides
    elif layout == "bthd":
        NB, bs, H, D = shape
        s_blk, s_t, s_h, s_d = strides
    else:
        raise ValueError(f"unknown pool layout {layout!r}")
    if sc_shape != (NB, H, bs):
        raise ValueError(f"scale pool {tuple(sc_shape)} does not match pool {tuple(shape)}")
    sc_blk, sc_h, sc_t = sc_strides
    if s_d != 1 or sc_t != 1:
        raise ValueError("dims and scale tokens must be contiguous")
    if v_pool.stride() != strides or vs_pool.stride() != sc_strides or v_pool.shape != shape or vs_pool.shape != sc_shape:
        raise ValueError("K/V pools and their scale pools must share shapes and strides")
    for t in (k_pool, v_pool, ks_pool, vs_pool):
        if t.get_device() != device:
            raise _elsewhere(t)
    if k_pool.dtype is not i8 or v_pool.dtype is not i8 or ks_pool.dtype is not f32 or vs_pool.dtype is not f32:
        raise ValueError("pools are int8, scale pools float32")
    return NB, H, bs, D, s_blk, s_h, s_t, sc_blk, sc_h


def _table(device: int, block_table, B: int, i32) -> int:
    """Entries per row of an int32 [B, max_blocks] table."""
    shape = block_table.shape
    if block_table.dtype != i32 or len(shape) != 2 or shape[0] != B or block_table.stride(1) != 1:
        raise ValueError("block_table must be int32 [B, max_blocks] with contiguous rows")
    if block_table.get_device() != device:
        raise _elsewhere(block_table)
    return shape[1]


def paged_plan(seq_lens, new_lens, block_table, free_blocks, free_count, block_size: int, slot_map, token_starts=None,
               seq_lens_out=None, free_count_out=None, workspace=None, stream=None):
    """Block tables and slot maps from request lengths (``kvd_paged_plan_launch``).

    ``seq_lens`` / ``new_lens`` int32 [B] (tokens held, tokens to add; new_lens < 0 ends a request),
    ``block_table`` int32 [B, max_blocks], ``free_blocks`` int32 [num_blocks] with ``free_count`` int32 [1]
    ids on it, ``slot_map`` int64 [num_slots]. The table, the free list and, unless other tensors are given for
    them, the lengths and the count are updated in place. An ended request gives all its blocks back; requests that
    share blocks are ended by :func:`paged_fork`. ``workspace``: a zeroed uint8 tensor of 16 bytes that a
    caller keeps (without one, one is made). Returns (slot_map, token_starts [B + 1])."""
    torch, _, i32, i64, _ = _torch or _types()
    device, B = seq_lens.get_device(), seq_lens.shape[0]
    MB = _table(device, block_table, B, i32)
    NB, T = free_blocks.numel(), slot_map.numel()
    rows, one = (B,), (1,)
    _want(device, i32, (seq_lens, rows, "seq_lens"), (new_lens, rows, "new_lens"), (free_blocks, (NB,), "free_blocks"),
          (free_count, one, "free_count"), (token_starts, (B + 1,), "token_starts"),
          (seq_lens_out, rows, "seq_lens_out"), (free_count_out, one, "free_count_out"))
    _want(device, i64, (slot_map, (T,), "slot_map"))
    _own_scratch(device, workspace)
    handle = _handle(device, stream)
    if seq_lens_out is None:
        seq_lens_out = seq_lens
    if free_count_out is None:
        free_count_out = free_count
    if token_starts is None:
        token_starts = _out((B + 1,), i32, seq_lens, stream)
    if workspace is None:  # zeroed on the call's stream
        workspace = _made(torch.zeros, 16, torch.uint8, seq_lens, stream)
    desc = PagedPlanDesc(B, block_size, NB, MB, T, block_table.stride(0))
    rc = (_lib or lib()).kvd_paged_plan_launch(
        ctypes.byref(desc), seq_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(), free_blocks.data_ptr(),
        free_count.data_ptr(), slot_map.data_ptr(), token_starts.data_ptr(), seq_lens_out.data_ptr(),
        free_count_out.data_ptr(), workspace.data_ptr(), workspace.nbytes, handle)
    if rc:
        _check(rc, "kvd_paged_plan_launch")
    return slot_map, token_starts


def _rows_desc(device: int, k, v, slot_map, k_pool, v_pool, ks_pool, vs_pool, layout: str):
    NB, H, bs, D, s_blk, s_h, s_t, sc_blk, sc_h = _pools(device, k_pool, v_pool, ks_pool, vs_pool, layout)
    T, (s_row, s_head, s_dim) = slot_map.shape[0], k.stride()
    if k.shape != (T, H, D) or v.shape != k.shape or v.dtype != k.dtype or v.stride() != (s_row, s_head, s_dim) or s_dim != 1:
        raise ValueError(f"rows must be two [{T}, {H}, {D}] tensors of one type and strides with contiguous dims")
    _want(device, _torch[3], (slot_map, (T,), "slot_map"))
    if k.get_device() != device or v.get_device() != device:
        raise _elsewhere(v if k.get_device() == device else k)
    return PagedRowsDesc(T, H, D, bs, NB, _row_flags(k.dtype), s_row, s_head, s_blk, s_h, s_t, sc_blk, sc_h)


def paged_write(k_new, v_new, slot_map, k_pool, v_pool, ks_pool, vs_pool, bounds=None, bound_scale=None,
                layout: str = "bhtd", stream=None) -> None:
    """Quantises rows k_new / v_new [T, Hkv, D] (float32, bfloat16 or float16) into the pools' slots
    ``slot_map`` [T] (-1: skipped). With ``bounds`` int8 [blocks, Hkv, 2, D] and ``bound_scale`` float32
    [blocks, Hkv] the key bounds of every block written to are kept for :func:`block_select`."""
    device = k_pool.get_device()
    desc = _rows_desc(device, k_new, v_new, slot_map, k_pool, v_pool, ks_pool, vs_pool, layout)
    if (bounds is None) != (bound_scale is None):
        raise ValueError("bounds and bound_scale come together")
    bounds_ptr = scale_ptr = None
    if bounds is not None:
        NB, H = desc.num_blocks, desc.num_kv_heads
        _want(device, _torch[1], (bounds, (NB, H, 2, desc.head_dim), "bounds"))
        _want(device, _torch[4], (bound_scale, (NB, H), "bound_scale"))
        bounds_ptr, scale_ptr = bounds.data_ptr(), bound_scale.data_ptr()
    rc = (_lib or lib()).kvd_paged_write_launch(
        ctypes.byref(desc), k_new.data_ptr(), v_new.data_ptr(), slot_map.data_ptr(), k_pool.data_ptr(),
        v_pool.data_ptr(), ks_pool.data_ptr(), vs_pool.data_ptr(), bounds_ptr, scale_ptr, _handle(device, stream))
    if rc:
        _check(rc, "kvd_paged_write_launch")


def paged_read(slot_map, k_pool, v_pool, ks_pool, vs_pool, k_out=None, v_out=None, layout: str = "bhtd", dtype=None,
               stream=None):
    """Rows of a paged cache by slot as the values that they stand for: returns (k_out, v_out) [T, Hkv, D]
    (``dtype``, default float32; an output that is given sets the type and strides of the other). Slots of -1 read as
    zeros."""
    device = k_pool.get_device()
    handle = _handle(device, stream)
    if k_out is None and v_out is None:
        H, D = k_pool.shape[1 if layout == "bhtd" else 2], k_pool.shape[3]
        shape = (slot_map.shape[0], H, D)
        k_out, v_out = (_out(shape, dtype, k_pool, stream) for _ in range(2))
    else:
        given = v_out if k_out is None else k_out
        if dtype is not None and given.dtype is not dtype:
            raise ValueError(f"outputs of {given.dtype} are given, {dtype} is asked for")
        if k_out is None or v_out is None:
            make = lambda shape, **how: (_torch or _types())[0].empty_strided(shape, given.stride(), **how)  # noqa: E731
            other = _made(make, given.shape, given.dtype, k_pool, stream, True)
            k_out, v_out = (other, v_out) if k_out is None else (k_out, other)
    desc = _rows_desc(device, k_out, v_out, slot_map, k_pool, v_pool, ks_pool, vs_pool, layout)
    rc = (_lib or lib()).kvd_paged_read_launch(
        ctypes.byref(desc), slot_map.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), ks_pool.data_ptr(),
        vs_pool.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), handle)
    if rc:
        _check(rc, "kvd_paged_read_launch")
    return k_out, v_out


def block_select(q, bounds, bound_scale, block_table, seq_lens, block_size: int, budget: int, first: int = 1,
                 last: int = 2, sel_table=None, sel_lens=None, workspace=None, stream=None):
    """Blocks that one new token per request attends to (``kvd_block_select_launch``): the ``first`` first and
    ``last`` last blocks and those whose key bounds score highest for ``q`` [B, Hq, D], ``budget`` in all, per
    KV head. Returns (sel_table int32 [B, Hkv, budget] pool ids, then -1; sel_lens int32 [B, Hkv] tokens)."""
    torch, i8, i32, _, f32 = _torch or _types()
    B, Hq, D = q.shape
    NB, H, _, Db = bounds.shape
    if Db != D or Hq % H:
        raise ValueError(f"shape mismatch q{tuple(q.shape)} bounds{tuple(bounds.shape)}")
    s_b, s_h, s_d = q.stride()
    if s_d != 1:
        raise ValueError("dims must be contiguous")
    device = q.get_device()
    MB = _table(device, block_table, B, i32)
    _want(device, i8, (bounds, (NB, H, 2, D), "bounds"))
    _want(device, f32, (bound_scale, (NB, H), "bound_scale"))
    _want(device, i32, (seq_lens, (B,), "seq_lens"), (sel_table, (B, H, budget), "sel_table"),
          (sel_lens, (B, H), "sel_lens"))
    _own_scratch(device, workspace)
    handle = _handle(device, stream)
    if sel_table is None:
        sel_table = _out((B, H, budget), i32, q, stream)
    if sel_lens is None:
        sel_lens = _out((B, H), i32, q, stream)
    desc = BlockSelectDesc(B, Hq, H, D, block_size, NB, MB, budget, first, last, _row_flags(q.dtype),
                           seq_lens.data_ptr(), block_table.data_ptr(), block_table.stride(0), s_b, s_h)
    if workspace is None and MB > budget:
        workspace = _scratch(B * H * MB * 4, q, stream)
    rc = (_lib or lib()).kvd_block_select_launch(
        ctypes.byref(desc), q.data_ptr(), bounds.data_ptr(), bound_scale.data_ptr(), sel_table.data_ptr(),
        sel_lens.data_ptr(), _ptr(workspace), workspace.nbytes if workspace is not None else 0, handle)
    if rc:
        _check(rc, "kvd_block_select_launch")
    return sel_table, sel_lens


def sparse_workspace_size(q, k_pool, sel_table, layout: str = "bhtd") -> int:
    """Bytes of scratch :func:`sparse_decode` uses for these shapes."""
    B, Hq, D = q.shape
    NB, H, bs = (k_pool.shape[i] for i in ((0, 1, 2) if layout == "bhtd" else (0, 2, 1)))
    p = sel_table.data_ptr()
    desc = PagedDesc(B, Hq, H, D, bs, NB, sel_table.shape[-1], 0, p, p, sel_table.shape[-1])
    return int(lib().kvd_sparse_workspace_size(ctypes.byref(desc)))


def sparse_decode(q, k_pool, v_pool, ks_pool, vs_pool, sel_table, sel_lens, out=None, layout: str = "bhtd",
                  softmax_scale: float = 0.0, partial: bool = False, workspace=None, stream=None, out_dtype=None):
    """INT8 decode attention over selected blocks of a paged cache, ``sel_table`` int32 [B, Hkv, budget] and
    ``sel_lens`` int32 [B, Hkv] (:func:`block_select`'s); returns ``out`` [B, Hq, D] (or records)."""
    torch, _, i32, _, f32 = _torch or _types()
    B, Hq, D = q.shape
    R = D + 4 if partial else D
    if out is not None and out.shape != (B, Hq, R):
        raise ValueError(f"out must be [{B}, {Hq}, {R}], got {tuple(out.shape)}")
    device = q.get_device()
    NB, H, bs, Dk, s_blk, s_h, s_t, sc_blk, sc_h = _pools(device, k_pool, v_pool, ks_pool, vs_pool, layout)
    if Dk != D or Hq % H:
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k_pool{tuple(k_pool.shape)}")
    budget = sel_table.shape[-1]
    _want(device, i32, (sel_table, (B, H, budget), "sel_table"), (sel_lens, (B, H), "sel_lens"))
    if out is not None and out.get_device() != device:
        raise _elsewhere(out)
    _own_scratch(device, workspace)
    handle = _handle(device, stream)
    if out is None:
        out = _out((B, Hq, R), out_dtype, q, stream)
    q_b, q_h, q_d = q.stride()
    o_b, o_h, o_d = out.stride()
    if q_d != 1 or o_d != 1:
        raise ValueError("dims must be contiguous")
    if partial and out.dtype is not f32:
        raise ValueError("partial records are float32")
    flags = _row_flags(q.dtype) | _row_flags(out.dtype) << 2 | (KVD_FLAG_PARTIAL_OUT if partial else 0)  # OUT_*: two bits up
    table = sel_table.data_ptr()
    desc = PagedDesc(B, Hq, H, D, bs, NB, budget, flags, sel_lens.data_ptr(), table, budget,
                     s_blk, s_h, s_t, sc_blk, sc_h, q_b, q_h, o_b, o_h, softmax_scale)
    if workspace is None:
        n = int(lib().kvd_sparse_workspace_size(ctypes.byref(desc)))
        workspace = _scratch(n, q, stream)
    rc = (_lib or lib()).kvd_sparse_decode_launch(
        ctypes.byref(desc), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), ks_pool.data_ptr(), vs_pool.data_ptr(),
        out.data_ptr(), workspace.data_ptr(), workspace.nbytes, handle)
    if rc:
        _check(rc, "kvd_sparse_decode_launch")
    return out


def _prefill_desc(q, k_pool, block_table, layout: str, causal: bool = True):
    """Descriptor of the sizes alone, for the workspace."""
    T, Hq, D = q.shape
    NB, H, bs = (k_pool.shape[i] for i in ((0, 1, 2) if layout == "bhtd" else (0, 2, 1)))
    B, MB = block_table.shape
    p = block_table.data_ptr() or 16
    desc = PagedPrefillDesc(B, Hq, H, D, T, bs, NB, MB, int(causal), _row_flags(q.dtype), p, p, p, MB)
    return desc


def paged_prefill_workspace_size(q, k_pool, block_table, layout: str = "bhtd") -> int:
    """Bytes of scratch :func:`paged_prefill` uses for these shapes. They do not fall as ``q`` gets rows, so scratch for a
    loop's largest step serves the others."""
    return int(lib().kvd_paged_prefill_workspace_size(ctypes.byref(_prefill_desc(q, k_pool, block_table, layout))))


def paged_prefill(q, k_pool, v_pool, ks_pool, vs_pool, block_table, seq_lens, token_starts, out=None, layout: str = "bhtd",
                  causal: bool = True, softmax_scale: float = 0.0, workspace=None, stream=None, out_dtype=None):
    """Attention of the new tokens of every request over a paged INT8 cache (``kvd_paged_prefill_launch``).

    ``q`` [T, Hq, D] (float32, bfloat16 or float16) holds the requests' rows one after the other, request b's from
    ``token_starts``[b] to ``token_starts``[b + 1] (int32 [B + 1], :func:`paged_plan`'s), any number of them, single
    tokens among them. They are the last of its ``seq_lens``[b] tokens, whose K/V rows the cache holds already; each
    attends to the tokens up to its own, or with ``causal=False`` to all of them (an encoder's states). Returns ``out``
    [T, Hq, D]; rows that belong to no request are left as they are."""
    torch, _, i32, _, _ = _torch or _types()
    T, Hq, D = q.shape
    device = q.get_device()
    NB, H, bs, Dk, s_blk, s_h, s_t, sc_blk, sc_h = _pools(device, k_pool, v_pool, ks_pool, vs_pool, layout)
    if Dk != D or Hq % H:
        raise ValueError(f"shape mismatch q{tuple(q.shape)} k_pool{tuple(k_pool.shape)}")
    B = seq_lens.shape[0]
    MB = _table(device, block_table, B, i32)
    _want(device, i32, (seq_lens, (B,), "seq_lens"), (token_starts, (B + 1,), "token_starts"))
    if out is not None:
        if out.shape != (T, Hq, D):
            raise ValueError(f"out must be [{T}, {Hq}, {D}], got {tuple(out.shape)}")
        if out.get_device() != device:
            raise _elsewhere(out)
        if out_dtype is not None and out.dtype is not out_dtype:
            raise ValueError(f"an output of {out.dtype} is given, {out_dtype} is asked for")
    _own_scratch(device, workspace)
    handle = _handle(device, stream)
    if out is None:
        out = _out((T, Hq, D), out_dtype, q, stream)
    q_t, q_h, q_d = q.stride()
    o_t, o_h, o_d = out.stride()
    if q_d != 1 or o_d != 1:
        raise ValueError("dims must be contiguous")
    flags = _row_flags(q.dtype) | _row_flags(out.dtype) << 2  # KVD_FLAG_OUT_* lie two bits above KVD_FLAG_Q_*
    desc = PagedPrefillDesc(B, Hq, H, D, T, bs, NB, MB, 1 if causal else 0, flags, seq_lens.data_ptr(),
                            token_starts.data_ptr(), block_table.data_ptr(), block_table.stride(0), s_blk, s_h, s_t,
                            sc_blk, sc_h, q_t, q_h, o_t, o_h, softmax_scale)
    if workspace is None:
        workspace = _scratch(int(lib().kvd_paged_prefill_workspace_size(ctypes.byref(desc))), q, stream)
    rc = (_lib or lib()).kvd_paged_prefill_launch(
        ctypes.byref(desc), q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), ks_pool.data_ptr(), vs_pool.data_ptr(),
        out.data_ptr(), workspace.data_ptr(), workspace.nbytes, handle)
    if rc:
        _check(rc, "kvd_paged_prefill_launch")
    return out


def _pages_desc(device: int, seq_lens, block_table, block_table_out, free_blocks, free_count, k_pool, v_pool, ks_pool,
                vs_pool, bounds, bound_scale, layout: str, i32, i8, f32):
    """Checked descriptor of a call on whole blocks."""
    NB, H, bs, D, s_blk, s_h, s_t, sc_blk, sc_h = _pools(device, k_pool, v_pool, ks_pool, vs_pool, layout)
    B = seq_lens.shape[0]
    MB = _table(device, block_table, B, i32)
    if block_table_out is not block_table and _table(device, block_table_out, B, i32) != MB:
        raise ValueError(f"block_table_out must be [{B}, {MB}], got {tuple(block_table_out.shape)}")
    if (bounds is None) != (bound_scale is None):
        raise ValueError("bounds and bound_scale come together")
    _want(device, i32, (seq_lens, (B,), "seq_lens"), (free_blocks, (NB,), "free_blocks"), (free_count, (1,), "free_count"))
    _want(device, i8, (bounds, (NB, H, 2, D), "bounds"))
    _want(device, f32, (bound_scale, (NB, H), "bound_scale"))
    return PagesDesc(B, H, D, bs, NB, MB, block_table.stride(0), block_table_out.stride(0), s_blk, s_h, s_t, sc_blk, sc_h)


def _pages_size(name: str, block_table, free_blocks) -> int:
    B, MB = block_table.shape
    desc = PagesDesc(B, 1, 1, 1, free_blocks.numel(), MB, MB, MB)
    return int(getattr(lib(), name)(ctypes.byref(desc)))


def paged_fork_workspace_size(block_table, free_blocks) -> int:
    """Bytes of zeroed scratch that :func:`paged_fork` keeps between calls for these shapes."""
    return _pages_size("kvd_paged_fork_workspace_size", block_table, free_blocks)


def paged_compact_workspace_size(block_table, free_blocks) -> int:
    """Bytes of zeroed scratch that :func:`paged_compact` keeps between calls for these shapes."""
    return _pages_size("kvd_paged_compact_workspace_size", block_table, free_blocks)


def paged_fork(parents, seq_lens, block_table, free_blocks, free_count, k_pool, v_pool, ks_pool, vs_pool, bounds=None,
               bound_scale=None, layout: str = "bhtd", seq_lens_out=None, block_table_out=None, free_count_out=None,
               workspace=None, stream=None):
    """Rows of the block table become copies of other rows (``kvd_paged_fork_launch``): row b continues row
    ``parents``[b] (int32 [B]; b itself: it goes on as it is; -1: it ends). Full blocks are shared, partly filled
    last ones are copied into blocks from the free list, and blocks that no row names any more go back on it.
    Lengths, table and count are updated in place unless other tensors are given for them (as for all layers but
    the last where several share a table). Requests that may share blocks are ended here, not by
    :func:`paged_plan`. A length that is lowered by hand (refused drafts) stays inside a last block that no other row
    names: blocks behind it are lost to the pool, and a shared one that it ends in would be written to. ``workspace``: a zeroed uint8 tensor of :func:`paged_fork_workspace_size` bytes that a
    caller keeps for pools of as many blocks (without one, one is made). Returns (block_table_out, seq_lens_out)."""
    torch, i8, i32, _, f32 = _torch or _types()
    device = seq_lens.get_device()
    if block_table_out is None:
        block_table_out = block_table
    desc = _pages_desc(device, seq_lens, block_table, block_table_out, free_blocks, free_count, k_pool, v_pool, ks_pool,
                       vs_pool, bounds, bound_scale, layout, i32, i8, f32)
    rows = (desc.batch,)
    _want(device, i32, (parents, rows, "parents"), (seq_lens_out, rows, "seq_lens_out"),
          (free_count_out, (1,), "free_count_out"))
    _own_scratch(device, workspace)
    handle = _handle(device, stream)
    if seq_lens_out is None:
        seq_lens_out = seq_lens
    if free_count_out is None:
        free_count_out = free_count
    if workspace is None:  # zeroed on the call's stream
        n = int(lib().kvd_paged_fork_workspace_size(ctypes.byref(desc)))
        workspace = _made(torch.zeros, n or 1, torch.uint8, seq_lens, stream)
    rc = (_lib or lib()).kvd_paged_fork_launch(
        ctypes.byref(desc), parents.data_ptr(), seq_lens.data_ptr(), block_table.data_ptr(), free_blocks.data_ptr(),
        free_count.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), ks_pool.data_ptr(), vs_pool.data_ptr(), _ptr(bounds),
        _ptr(bound_scale), seq_lens_out.data_ptr(), block_table_out.data_ptr(), free_count_out.data_ptr(),
        workspace.data_ptr(), workspace.nbytes, handle)
    if rc:
        _check(rc, "kvd_paged_fork_launch")
    return block_table_out, seq_lens_out


def paged_compact(seq_lens, block_table, free_blocks, free_count, k_pool, v_pool, ks_pool, vs_pool, bounds=None,
                  bound_scale=None, layout: str = "bhtd", block_table_out=None, free_blocks_out=None, used=None,
                  workspace=None, stream=None):
    """Moves the blocks that the table names to the lowest ids among those and the free ones
    (``kvd_paged_compact_launch``). Table and free list are updated in place unless other tensors are given for
    them, ``free_count`` always is. ``workspace``: a zeroed uint8 tensor of :func:`paged_compact_workspace_size`
    bytes that a caller keeps. Returns ``used`` int32 [1]: the blocks that the pools then need."""
    torch, i8, i32, _, f32 = _torch or _types()
    device = seq_lens.get_device()
    if block_table_out is None:
        block_table_out = block_table
    if free_blocks_out is None:
        free_blocks_out = free_blocks
    desc = _pages_desc(device, seq_lens, block_table, block_table_out, free_blocks, free_count, k_pool, v_pool, ks_pool,
                       vs_pool, bounds, bound_scale, layout, i32, i8, f32)
    _want(device, i32, (free_blocks_out, (desc.num_blocks,), "free_blocks_out"), (used, (1,), "used"))
    _own_scratch(device, workspace)
    handle = _handle(device, stream)
    if used is None:
        used = _out((1,), i32, seq_lens, stream)
    if workspace is None:  # zeroed on the call's stream
        n = int(lib().kvd_paged_compact_workspace_size(ctypes.byref(desc)))
        workspace = _made(torch.zeros, n or 1, torch.uint8, seq_lens, stream)
    rc = (_lib or lib()).kvd_paged_compact_launch(
        ctypes.byref(desc), seq_lens.data_ptr(), block_table.data_ptr(), free_blocks.data_ptr(), free_count.data_ptr(),
        k_pool.data_ptr(), v_pool.data_ptr(), ks_pool.data_ptr(), vs_pool.data_ptr(), _ptr(bounds), _ptr(bound_scale),
        block_table_out.data_ptr(), free_blocks_out.data_ptr(), used.data_ptr(), workspace.data_ptr(), workspace.nbytes,
        handle)
    if rc:
        _check(rc, "kvd_paged_compact_launch")
    return used


# ------------------------------------------------------------------ multi-GPU
def mgpu_unique_id() -> bytes:
    """A fresh 128-byte NCCL unique id (made on one rank, broadcast by the caller)."""
    buf = (ctypes.c_ubyte * 128)()
    rc = lib().kvd_mgpu_get_unique_id(ctypes.addressof(buf))
    if rc != 0:
        raise RuntimeError(f"kvd_mgpu_get_unique_id failed: nccl error {rc}")
    return bytes(buf)


class MgpuComm:
    """An NCCL communicator made by the library (kvd_mgpu_comm_init)."""

    def __init__(self, nranks: int, rank: int, uid: bytes):
        buf = (ctypes.c_ubyte * 128).from_buffer_copy(uid)
        h = c_void_p()
        rc = lib().kvd_mgpu_comm_init(ctypes.byref(h), nranks, rank, ctypes.addressof(buf))
        if rc != 0:
            raise RuntimeError(f"kvd_mgpu_comm_init failed: nccl error {rc}")
        self.handle, self.nranks, self.rank = h.value, nranks, rank

    def close(self) -> None:
        if self.handle:
            lib().kvd_mgpu_comm_destroy(self.handle)
            self.handle = None


def seq_split_decode(comm: MgpuComm, q, k, v, ks, vs, out=None, seq_lens=None, workspace=None, stream=None,
                     out_dtype=None):
    """Sequence-split decode (kvd_mgpu_seq_split_decode): this rank passes its own token
    range of the cache; every rank gets the merged output rows."""
    B, Hq, D = q.shape
    if out is None:
        out = _out((B, Hq, D), out_dtype, q, stream)
    desc = make_desc(q, k, ks, out, seq_lens)
    if workspace is None:
        n = int(lib().kvd_mgpu_seq_split_workspace_size(ctypes.byref(desc), comm.nranks))
        workspace = _scratch(n, q, stream)
    rc = lib().kvd_mgpu_seq_split_decode(ctypes.byref(desc), _ptr(q), _ptr(k), _ptr(v), _ptr(ks), _ptr(vs),
                                         _ptr(out), _ptr(workspace), workspace.numel(), comm.handle, comm.nranks,
                                         _stream(stream))
    _check(rc, "kvd_mgpu_seq_split_decode")
    return out


class P2PExchange:
    """Sequence-split exchange over NVLink peer stores (kvd_mgpu_p2p_*); collective to create."""

    def __init__(self, comm: MgpuComm, batch: int, num_q_heads: int, head_dim: int):
        h = c_void_p()
        _check(lib().kvd_mgpu_p2p_create(ctypes.byref(h), batch, num_q_heads, head_dim, comm.handle, comm.nranks,
                                         comm.rank), "kvd_mgpu_p2p_create")
        self.handle = h.value
        self._ws = None

    def decode(self, q, k, v, ks, vs, out=None, seq_lens=None, stream=None, out_dtype=None):
        B, Hq, D = q.shape
        if out is None:
            out = _out((B, Hq, D), out_dtype, q, stream)
        desc = make_desc(q, k, ks, out, seq_lens)
        n = int(lib().kvd_mgpu_p2p_workspace_size(ctypes.byref(desc)))
        if self._ws is None or self._ws.numel() < n:
            self._ws = _scratch(n, q, stream)
        rc = lib().kvd_mgpu_p2p_seq_split_decode(self.handle, ctypes.byref(desc), _ptr(q), _ptr(k), _ptr(v),
                                                 _ptr(ks), _ptr(vs), _ptr(out), _ptr(self._ws), self._ws.numel(),
                                                 _stream(stream))
        _check(rc, "kvd_mgpu_p2p_seq_split_decode")
        return out

    def reset(self, stream=None) -> None:
        """Collective: clears the exchange state on every rank after a call timed
        out (KVD_STATUS_WAIT_TIMEOUT), so the ranks' calls pair up again."""
        _check(lib().kvd_mgpu_p2p_reset(self.handle, _stream(stream)), "kvd_mgpu_p2p_reset")

    def close(self) -> None:
        if self.handle:
            lib().kvd_mgpu_p2p_destroy(self.handle)
            self.handle = None


class P2PGroup:
    """Single-process sequence split (kvd_mgpu_p2p_create_group): one context per
    rank, rank r on device devices[r], linked by direct peer pointers."""

    def __init__(self, devices, batch: int, num_q_heads: int, head_dim: int):
        n = len(devices)
        hs = (c_void_p * n)()
        devs = (c_int * n)(*devices)
        _check(lib().kvd_mgpu_p2p_create_group(hs, n, devs, batch, num_q_heads, head_dim),
               "kvd_mgpu_p2p_create_group")
        self.handles = [hs[r] for r in range(n)]
        self.devices = list(devices)
        self._ws = {}

    def decode(self, rank: int, q, k, v, ks, vs, out=None, seq_lens=None, stream=None, out_dtype=None):
        """Launches rank `rank`'s step on its device (tensors on that device); returns without waiting."""
        import torch

        with torch.cuda.device(self.devices[rank]):
            B, Hq, D = q.shape
            if out is None:
                out = _out((B, Hq, D), out_dtype, q, stream)
            desc = make_desc(q, k, ks, out, seq_lens)
            n = int(lib().kvd_mgpu_p2p_workspace_size(ctypes.byref(desc)))
            ws = self._ws.get(rank)
            if ws is None or ws.numel() < n:
                ws = self._ws[rank] = _scratch(n, q, stream)
            rc = lib().kvd_mgpu_p2p_seq_split_decode(self.handles[rank], ctypes.byref(desc), _ptr(q), _ptr(k),
                                                     _ptr(v), _ptr(ks), _ptr(vs), _ptr(out), _ptr(ws), ws.numel(),
                                                     _stream(stream))
        _check(rc, "kvd_mgpu_p2p_seq_split_decode")
        return out

    def reset(self) -> None:
        for h in self.handles:
            _check(lib().kvd_mgpu_p2p_reset(h, None), "kvd_mgpu_p2p_reset")

    def close(self) -> None:
        for h in self.handles:
            if h:
                lib().kvd_mgpu_p2p_destroy(h)
        self.handles = []


def device_status() -> int:
    """Synchronise, then read and clear the device status word (KVD_STATUS_* bits)."""
    v = c_int32(0)
    _check(lib().kvd_device_status(ctypes.byref(v)), "kvd_device_status")
    return int(v.value)


def last_launch_count() -> int:
    return int(lib().kvd_last_launch_count())


def algorithmic_bytes(B: int, Hq: int, Hkv: int, D: int, lens) -> int:
    """Bytes a decode step must move: each (b, kv head) reads its codes and two
    scales per token once, plus the fp32 query and output rows."""
    if isinstance(lens, int):
        tokens = B * lens
    else:
        tokens = int(sum(int(x) for x in lens))
    return tokens * Hkv * (2 * D + 8) + B * Hq * D * 4 * 2


def default_softmax_scale(D: int) -> float:
    return 1.0 / math.sqrt(D)
