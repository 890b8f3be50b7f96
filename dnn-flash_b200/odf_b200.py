"""Python binding of the C ABI in include/odf_sm100.h (ctypes; torch tensors for device memory).

This module adds no compute of its own: every call goes through
``lib/libodf_sm100.so``.  If that library is missing the import fails loudly;
there is no CPU fallback.  Argument meaning and error behaviour follow the
reference's batched entry point ``flash_attention_batched_qk_pv_tile``
(src/onednn_flash/batched_attention.cpp:9-49): invalid sizes or null tensors
raise ``ValueError`` (the reference's ``std::invalid_argument``), anything the
GPU path cannot run raises ``RuntimeError`` (its ``std::runtime_error``).
"""
from __future__ import annotations

import ctypes as C
import math
import operator
import os
import struct
from pathlib import Path

PACKAGE_DIR = Path(__file__).resolve().parent
LIB_PATH = PACKAGE_DIR / "lib" / "libodf_sm100.so"
HEADER_PATHS = sorted((PACKAGE_DIR.parent / "include").glob("*.h"))

ODF_OK = 0
ODF_ERR_INVALID_ARG = 1
ODF_ERR_UNSUPPORTED = 2
ODF_ERR_CUDA = 3
ODF_ERR_DEVICE_TIMEOUT = 4
ODF_ERR_NO_DEVICE = 5
ODF_ERR_BAD_PAGE = 7
ODF_ERR_NO_PAGES = 8
ODF_DTYPE_F32 = 0
ODF_DTYPE_BF16 = 1
ODF_DTYPE_E4M3 = 16
ODF_BIAS_NONE = 0
ODF_BIAS_SAME_SHAPE = 1
ODF_BIAS_ALIBI = 4
TILE_Q = 128
TILE_K = 128
_INT64_MAX = 2 ** 63 - 1


class FwdParams(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("o", C.c_void_p), ("lse", C.c_void_p),
        ("qkv_dtype", C.c_int32), ("o_dtype", C.c_int32),
        ("batch", C.c_int64), ("heads_q", C.c_int64), ("heads_kv", C.c_int64),
        ("seqlen_q", C.c_int64), ("seqlen_k", C.c_int64), ("head_dim", C.c_int64), ("value_dim", C.c_int64),
        ("q_strides", C.c_int64 * 3), ("k_strides", C.c_int64 * 3), ("v_strides", C.c_int64 * 3),
        ("o_strides", C.c_int64 * 3),
        ("scale", C.c_float), ("causal", C.c_int32),
        ("block_mask", C.c_void_p), ("mask_qbs", C.c_int64), ("mask_kbs", C.c_int64),
        ("mask_qblocks", C.c_int64), ("mask_kblocks", C.c_int64),
        ("bias_kind", C.c_int32), ("alibi_slopes", C.c_void_p), ("softcap", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("tile_visits", C.c_void_p),
        ("bias", C.c_void_p), ("bias_strides", C.c_int64 * 4),
    ]


class Window(C.Structure):
    _fields_ = [("window", C.c_int64), ("sinks", C.c_int64), ("q_offset", C.c_int64)]


class PagedCache(C.Structure):
    _fields_ = [
        ("k_pages", C.c_void_p), ("v_pages", C.c_void_p), ("kv_dtype", C.c_int32),
        ("num_pages", C.c_int64), ("heads_kv", C.c_int64), ("page_size", C.c_int64), ("head_dim", C.c_int64),
        ("k_strides", C.c_int64 * 3), ("v_strides", C.c_int64 * 3),
        ("k_scale", C.c_void_p), ("v_scale", C.c_void_p),
        ("page_table", C.c_void_p), ("table_stride", C.c_int64), ("max_pages", C.c_int64),
    ]


class DecodeParams(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("o", C.c_void_p), ("lse", C.c_void_p), ("o_dtype", C.c_int32),
        ("batch", C.c_int64), ("heads_q", C.c_int64), ("q_strides", C.c_int64 * 2), ("o_strides", C.c_int64 * 2),
        ("lens", C.c_void_p), ("cache", PagedCache), ("scale", C.c_float), ("window", C.c_int64),
        ("sinks", C.c_int64), ("bias_kind", C.c_int32), ("alibi_slopes", C.c_void_p), ("softcap", C.c_float),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class AppendParams(C.Structure):
    _fields_ = [
        ("k", C.c_void_p), ("v", C.c_void_p), ("batch", C.c_int64), ("tokens", C.c_int64),
        ("k_strides", C.c_int64 * 3), ("v_strides", C.c_int64 * 3),
        ("starts", C.c_void_p), ("counts", C.c_void_p), ("cache", PagedCache),
    ]


class PageCopyParams(C.Structure):
    _fields_ = [
        ("cache", PagedCache), ("layers", C.c_int64), ("k_layer_stride", C.c_int64), ("v_layer_stride", C.c_int64),
        ("pairs", C.c_void_p), ("n_pairs", C.c_int64),
    ]


# The same structs as one struct.pack call each, in field order (ctypes takes three times as long to
# build them, as long as a short kernel runs).
_CACHE_FORMAT = "PPi4q3q3qPPPqq"
_PACK_DECODE = struct.Struct("@PPPi2q2q2qP" + _CACHE_FORMAT + "fqqiPfPN").pack
_PACK_APPEND = struct.Struct("@PPqq3q3qPP" + _CACHE_FORMAT).pack
_PACK_COPY = struct.Struct("@" + _CACHE_FORMAT + "qqqPq").pack
_PACK_FWD = struct.Struct("@5Pii7q3q3q3q3qfiP4qiPfPNPP4q").pack
_PACK_WINDOW = struct.Struct("@qqq").pack


class OdfError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"odf status {code}: {message}")
        self.code = code


_lib = None


def load_library():
    """Load the sm_100a library (raises if it was not built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.exists():
        raise ImportError(f"{LIB_PATH} is missing: build it with __graft_entry__.build() (no CPU fallback exists)")
    lib = C.CDLL(str(LIB_PATH))
    lib.odf_flash_fwd_sm100.argtypes = [C.POINTER(FwdParams), C.c_void_p]
    lib.odf_flash_fwd_host.argtypes = [C.POINTER(FwdParams)]
    lib.odf_fwd_workspace_size.argtypes = [C.POINTER(FwdParams)]
    lib.odf_fwd_workspace_size.restype = C.c_size_t
    # c_void_p takes a packed struct (bytes), byref() of a ctypes one, or None
    lib.odf_flash_fwd_window_sm100.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p]
    lib.odf_fwd_window_workspace_size.argtypes = [C.c_void_p, C.c_void_p]
    lib.odf_fwd_window_workspace_size.restype = C.c_size_t
    lib.odf_tile_map_sm100.argtypes = [C.c_int64, C.c_int64, C.c_int32, C.c_void_p, C.c_int64, C.c_int64,
                                       C.c_int64, C.c_int64, C.c_void_p, C.c_void_p]
    lib.odf_convert_f32_to_bf16.argtypes = [C.c_void_p, C.c_void_p, C.c_int64, C.c_void_p]
    lib.odf_device_status.argtypes = [C.POINTER(C.c_int32), C.c_int32]
    lib.odf_paged_decode_sm100.argtypes = [C.c_void_p, C.c_void_p]
    lib.odf_paged_decode_workspace_size.argtypes = [C.c_void_p]
    lib.odf_paged_decode_workspace_size.restype = C.c_size_t
    lib.odf_paged_append_sm100.argtypes = [C.c_void_p, C.c_void_p]
    lib.odf_page_copy_sm100.argtypes = [C.c_void_p, C.c_void_p]
    i64, p64, p32 = C.c_int64, C.POINTER(C.c_int64), C.c_void_p
    lib.odf_page_pool_create.argtypes = [i64, i64, C.POINTER(C.c_void_p)]
    lib.odf_page_pool_destroy.argtypes = [C.c_void_p]
    lib.odf_page_pool_destroy.restype = None
    lib.odf_page_pool_add.argtypes = [C.c_void_p, p64]
    lib.odf_page_pool_fork.argtypes = [C.c_void_p, i64, p64]
    lib.odf_page_pool_extend.argtypes = [C.c_void_p, i64, i64, p32, p64]
    lib.odf_page_pool_truncate.argtypes = [C.c_void_p, i64, i64]
    lib.odf_page_pool_free.argtypes = [C.c_void_p, i64]
    lib.odf_page_pool_compact.argtypes = [C.c_void_p, p32, i64, p64]
    lib.odf_page_pool_length.argtypes = [C.c_void_p, i64, p64, p64]
    lib.odf_page_pool_table.argtypes = [C.c_void_p, i64, p32, i64]
    lib.odf_page_pool_free_pages.argtypes = [C.c_void_p]
    lib.odf_page_pool_free_pages.restype = i64
    lib.odf_last_error.restype = C.c_char_p
    lib.odf_version.restype = C.c_char_p
    _lib = lib
    return lib


def last_error() -> str:
    return load_library().odf_last_error().decode()


def version() -> str:
    return load_library().odf_version().decode()


def _check(rc: int):
    if rc == ODF_OK:
        return
    msg = last_error()
    if rc == ODF_ERR_INVALID_ARG:
        raise ValueError(f"odf status {rc}: {msg}")
    raise OdfError(rc, msg)


def declared_symbols() -> list[str]:
    """Every function name declared in include/*.h (the C ABI)."""
    import re

    names = []
    for path in HEADER_PATHS:
        text = path.read_text()
        text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
        for m in re.finditer(r"^\s*(?:const\s+)?[A-Za-z_][\w\s\*]*?\b(odf_\w+)\s*\(", text, flags=re.M):
            names.append(m.group(1))
    return sorted(set(names))


def alibi_slopes(heads: int) -> list[float]:
    """Generated ALiBi slopes 2^(-8 (h+1) / H), the values the kernel uses when none are given."""
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def _strides4(t):
    s = t.stride()
    if s[3] != 1:
        raise ValueError("the innermost (feature) dimension must be contiguous")
    if s[0] == s[1] == s[2] == 0 and max(t.shape[:3]) > 1:  # the C side would read zeros as a contiguous tensor's
        raise ValueError("q, k, v and out must not be broadcast (make them contiguous)")
    return (s[0], s[1], s[2])


def fill_params(q, k, v, o, lse, *, causal, scale, block_mask, mask_block, alibi, alibi_slopes_host, softcap,
                workspace, visits, bias=None) -> tuple[FwdParams, object]:
    """Populate odf_fwd_params from torch CUDA tensors; returns (params, keep-alive objects)."""
    import torch

    p = FwdParams()
    keep = []
    p.q, p.k, p.v, p.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr()
    p.lse = lse.data_ptr() if lse is not None else None
    p.qkv_dtype = ODF_DTYPE_BF16 if q.dtype == torch.bfloat16 else ODF_DTYPE_F32
    p.o_dtype = ODF_DTYPE_BF16 if o.dtype == torch.bfloat16 else ODF_DTYPE_F32
    B, Hq, M, D = q.shape
    _, Hkv, N, _ = k.shape
    p.batch, p.heads_q, p.heads_kv, p.seqlen_q, p.seqlen_k = B, Hq, Hkv, M, N
    p.head_dim, p.value_dim = D, v.shape[3]
    for name, t in (("q_strides", q), ("k_strides", k), ("v_strides", v), ("o_strides", o)):
        arr = getattr(p, name)
        for i, s in enumerate(_strides4(t)):
            arr[i] = s
    p.scale = scale
    p.causal = int(bool(causal))
    if block_mask is not None:
        p.block_mask = block_mask.data_ptr()
        p.mask_qbs, p.mask_kbs = mask_block
        p.mask_qblocks, p.mask_kblocks = block_mask.shape
    if alibi:
        p.bias_kind = ODF_BIAS_ALIBI
        if alibi_slopes_host is not None:
            arr = (C.c_float * len(alibi_slopes_host))(*[float(x) for x in alibi_slopes_host])
            keep.append(arr)
            p.alibi_slopes = C.cast(arr, C.c_void_p)
    p.softcap = softcap
    if bias is not None:
        if alibi:
            raise ValueError("ALiBi and a bias tensor are exclusive (one BiasKind per call)")
        # float32 CUDA tensor broadcastable to [B, Hq, M, N]; expand() gives 0 strides
        bias_v = bias.expand(B, Hq, M, N)
        strides = bias_v.stride()
        if not any(strides):  # one value for every score: all zero means contiguous on the C side, so a row of it
            bias_v, strides = bias_v[0, 0, 0].contiguous(), (0, 0, 0, 1)
        p.bias_kind = ODF_BIAS_SAME_SHAPE
        p.bias = bias_v.data_ptr()
        for i, st in enumerate(strides):
            p.bias_strides[i] = st
        keep.append(bias_v)
    if workspace is not None:
        p.workspace = workspace.data_ptr()
        p.workspace_bytes = workspace.numel() * workspace.element_size()
    if visits is not None:
        p.tile_visits = visits.data_ptr()
    return p, keep


def flash_fwd(q, k, v, *, causal=False, scale=None, block_mask=None, mask_block=(128, 128), alibi=False,
              alibi_slopes=None, softcap=0.0, out_dtype=None, want_lse=True, out=None, lse_out=None,
              visits=None, stream=None, bias=None):
    """Forward pass on CUDA tensors q [B,Hq,M,D], k [B,Hkv,N,D], v [B,Hkv,N,Dv] (bf16).

    ``bias``: optional float32 CUDA tensor broadcastable to [B,Hq,M,N], added after the
    scale (BiasKind::SameShapeTile).

    Returns (o [B,Hq,M,Dv], lse [B,Hq,M] fp32 natural log, or None).  The launch
    is asynchronous on ``stream`` (default: torch's current stream).
    """
    import torch

    lib = load_library()
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k, v must be rank 4 [B, H, T, D]")
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[3])
    B, Hq, M, _ = q.shape
    dev = q.device
    if out is None:
        out = torch.empty((B, Hq, M, v.shape[3]), dtype=out_dtype or torch.float32, device=dev)
    lse = lse_out
    if want_lse and lse is None:
        lse = torch.empty((B, Hq, M), dtype=torch.float32, device=dev)
    mask_t = None
    if block_mask is not None:
        mask_t = torch.as_tensor(block_mask, dtype=torch.uint8).to(dev).contiguous()
    p, keep = fill_params(q, k, v, out, lse, causal=causal, scale=scale, block_mask=mask_t, mask_block=mask_block,
                          alibi=alibi, alibi_slopes_host=alibi_slopes, softcap=softcap, workspace=None,
                          visits=visits, bias=bias)
    ws_bytes = lib.odf_fwd_workspace_size(C.byref(p))
    ws = None
    if ws_bytes:
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        p.workspace = ws.data_ptr()
        p.workspace_bytes = ws_bytes
    current = torch.cuda.current_stream(dev).cuda_stream
    if stream is None:
        stream = current
    bias_row = bias is not None and p.bias != bias.data_ptr()  # made above, on the current stream
    if bias_row and stream != current:
        torch.cuda.current_stream(dev).synchronize()
    _check(lib.odf_flash_fwd_sm100(C.byref(p), C.c_void_p(stream)))
    # Temporaries come from torch's allocator on the current stream; on another
    # stream they must outlive the launch, so wait for it before releasing them.
    if stream != current and (ws is not None or mask_t is not None or bias_row):
        torch.cuda.synchronize(dev)
    del keep
    return out, (lse if want_lse else None)


def flash_fwd_window(q, k, v, *, window, sinks=0, q_offset=0, scale=None, alibi=False, alibi_slopes=None, softcap=0.0,
                     out_dtype=None, want_lse=True, out=None, lse_out=None, stream=None):
    """Sliding-window attention with sinks (odf_flash_fwd_window_sm100) on q [B,Hq,M,D], k, v [B,Hkv,N,D] (bf16).

    Row i sits at position p = q_offset + i and sees key j iff j <= p and (p - j < window or j < sinks).
    ``q_offset``: tokens before this chunk of the prompt (0 for a whole one).  Returns (o, lse) like
    ``flash_fwd``, asynchronous on ``stream`` (default: torch's current stream).
    """
    import torch

    lib = load_library()
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("q must be [B, Hq, M, D], k and v of one shape [B, Hkv, N, D]")
    bf16 = torch.bfloat16
    if q.dtype is not bf16 or k.dtype is not bf16 or v.dtype is not bf16:
        raise ValueError("q, k and v must be bfloat16")
    B, Hq, M, D = q.shape
    dev = q.device
    _require_cuda(dev)
    _on(k, "k", dev)
    _on(v, "v", dev)
    slopes = _slopes_array(alibi_slopes, Hq) if alibi else None
    where, handle = _launch_on(dev, stream)
    with where:
        out, lse, o_code = _outputs(q, out, lse_out, out_dtype, want_lse, B, Hq, M)
        head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                ODF_DTYPE_BF16, o_code, B, Hq, k.shape[1], M, k.shape[2], D, D, *_strides(q, "q"), *_strides(k, "k"), *_strides(v, "v"), *_strides(out, "out"),
                1.0 / math.sqrt(D) if scale is None else scale, 1, 0, 0, 0, 0, 0,
                ODF_BIAS_ALIBI if alibi else ODF_BIAS_NONE, 0 if slopes is None else C.addressof(slopes), softcap)
        p = _PACK_FWD(*head, 0, 0, 0, 0, 0, 0, 0, 0)
        w = _PACK_WINDOW(_clip(window), _clip(sinks), _clip(q_offset))
        nbytes = lib.odf_fwd_window_workspace_size(p, w)
        if nbytes > 256:  # room for the parts of a split key range
            ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            p = _PACK_FWD(*head, ws.data_ptr(), nbytes, 0, 0, 0, 0, 0, 0)
        _check(lib.odf_flash_fwd_window_sm100(p, w, handle))
    return out, (lse if want_lse else None)


def flash_fwd_host(q, k, v, *, causal=False, scale=None, block_mask=None, mask_block=(128, 128), alibi=False,
                   alibi_slopes=None, softcap=0.0, out=None, lse_out=None, bias=None):
    """Forward pass on HOST numpy buffers through odf_flash_fwd_host (blocking).

    q/k/v are float32 or bfloat16-as-uint16 arrays [B,H,T,D]; ``out`` (float32 or
    uint16 for bf16) and ``lse_out`` (float32 [B,Hq,M] or None) are filled in place.
    """
    import numpy as np

    lib = load_library()
    B, Hq, M, D = q.shape
    _, Hkv, N, _ = k.shape
    p = FwdParams()
    p.q, p.k, p.v = q.ctypes.data, k.ctypes.data, v.ctypes.data
    p.qkv_dtype = ODF_DTYPE_F32 if q.dtype == np.float32 else ODF_DTYPE_BF16
    if out is None:
        out = np.empty((B, Hq, M, v.shape[3]), dtype=np.float32)
    p.o = out.ctypes.data
    p.o_dtype = ODF_DTYPE_F32 if out.dtype == np.float32 else ODF_DTYPE_BF16
    p.lse = lse_out.ctypes.data if lse_out is not None else None
    p.batch, p.heads_q, p.heads_kv, p.seqlen_q, p.seqlen_k, p.head_dim, p.value_dim = B, Hq, Hkv, M, N, D, v.shape[3]
    p.scale = (1.0 / math.sqrt(D)) if scale is None else scale
    p.causal = int(bool(causal))
    mask = None
    if block_mask is not None:
        mask = np.ascontiguousarray(block_mask, dtype=np.uint8)
        p.block_mask = mask.ctypes.data
        p.mask_qbs, p.mask_kbs = mask_block
        p.mask_qblocks, p.mask_kblocks = mask.shape
    keep = None
    if alibi:
        p.bias_kind = ODF_BIAS_ALIBI
        if alibi_slopes is not None:
            keep = (C.c_float * len(alibi_slopes))(*[float(x) for x in alibi_slopes])
            p.alibi_slopes = C.cast(keep, C.c_void_p)
    p.softcap = softcap
    bias_v = None
    if bias is not None:  # float32 array broadcastable to [B, Hq, M, N]
        bias_v = np.broadcast_to(np.asarray(bias, dtype=np.float32), (B, Hq, M, N))
        p.bias_kind = ODF_BIAS_SAME_SHAPE
        strides = [st // 4 for st in bias_v.strides]
        if not any(strides):  # one value for every score, as in fill_params
            bias_v, strides = np.ascontiguousarray(bias_v[0, 0, 0]), (0, 0, 0, 1)
        p.bias = bias_v.ctypes.data
        for i, st in enumerate(strides):
            p.bias_strides[i] = st
    _check(lib.odf_flash_fwd_host(C.byref(p)))
    del bias_v
    return out, lse_out


def tile_map(seqlen_q, seqlen_k, causal, block_mask=None, mask_block=(128, 128), device="cuda"):
    """Device tile map (uint8 [q_tiles, kv_tiles]: 0 skipped, 1 full, 2 element-masked)."""
    import torch

    lib = load_library()
    nqt, nkt = -(-seqlen_q // TILE_Q), -(-seqlen_k // TILE_K)
    out = torch.full((nqt, nkt), 255, dtype=torch.uint8, device=device)
    mask_t = None
    if block_mask is not None:
        mask_t = torch.as_tensor(block_mask, dtype=torch.uint8).to(device).contiguous()
        rc = lib.odf_tile_map_sm100(seqlen_q, seqlen_k, int(bool(causal)), mask_t.data_ptr(), mask_block[0],
                                    mask_block[1], mask_t.shape[0], mask_t.shape[1], out.data_ptr(),
                                    C.c_void_p(torch.cuda.current_stream().cuda_stream))
    else:
        rc = lib.odf_tile_map_sm100(seqlen_q, seqlen_k, int(bool(causal)), None, 0, 0, 0, 0, out.data_ptr(),
                                    C.c_void_p(torch.cuda.current_stream().cuda_stream))
    _check(rc)
    torch.cuda.synchronize()
    return out


# ------------------------------------------------------------------ paged key-value cache
# A decode step makes these calls once per layer, so they are written for few Python steps: structs are
# packed in one call, contiguous tensors pass zero strides, and the device and stream are only switched
# where they differ from the current ones.
_NO_STRIDES = (None, None, (0, 0), (0, 0, 0), (0, 0, 0))


def _strides(t, name):
    """Element strides of (up to three) dimensions before the last, which must be contiguous; all zero = contiguous."""
    n = t.dim() - 1
    if t.is_contiguous():
        return _NO_STRIDES[n]
    shape, stride = t.shape, t.stride()
    if n == 4:  # layers, which have a stride of their own
        n, shape, stride = 3, shape[1:], stride[1:]
    if stride[n] != 1:
        raise ValueError(f"the innermost (feature) dimension of {name} must be contiguous")
    out, dense = list(stride[:n]), shape[n]
    for i in range(n - 1, -1, -1):  # a dimension of size 1 has no stride of its own: a contiguous tensor's
        if shape[i] == 1:
            out[i] = dense
        elif out[i] == 0:  # with every dimension broadcast, the C side would read zeros as a contiguous tensor's
            raise ValueError(f"{name} is broadcast in dimension {i}, which the kernels do not take (make it contiguous)")
        dense *= shape[i]
    return out


def _on(tensor, name, device):
    if tensor.device != device:
        raise ValueError(f"{name} is on {tensor.device}, the call runs on {device}")


def _int32(tensor, name, device, rows):
    """Address of a contiguous int32 device vector of `rows` elements."""
    import torch

    if (tensor.dtype is not torch.int32 or tensor.shape != (rows,) or not tensor.is_contiguous()
            or tensor.device != device):
        _on(tensor, name, device)
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape [{rows}], got {tensor.dtype} {list(tensor.shape)}")
    return tensor.data_ptr()


def _scale_ptr(tensor, name, device, heads):
    import torch

    if tensor is None:
        return 0
    if tensor.dtype != torch.float32 or tensor.shape != (heads,) or not tensor.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 tensor [{heads}]")
    _on(tensor, name, device)
    return tensor.data_ptr()


def _cache_params(k_pages, v_pages, k_scale, v_scale, page_table, device, batch, heads=None, head_dim=None):
    """The values of odf_paged_cache for one layer's pages, checked against the call's other tensors.  Without
    a page table the pages may have a leading dimension of layers (page_copy)."""
    shape = k_pages.shape
    kind = _cache_kind(k_pages.dtype)
    if (kind is None or v_pages.dtype is not k_pages.dtype or v_pages.shape != shape or k_pages.device != device
            or v_pages.device != device or len(shape) not in (4, 5) or (len(shape) == 5 and page_table is not None)):
        raise _bad_cache(k_pages, v_pages, device)
    pages, hkv, page_size, dim = shape if len(shape) == 4 else shape[1:]
    if (heads is not None and heads != hkv) or (head_dim is not None and head_dim != dim):
        raise ValueError("the new tensors and the cache must have the same kv-heads and head_dim")
    table = table_stride = max_pages = 0
    if page_table is not None:
        rows, max_pages = page_table.shape if page_table.dim() == 2 else (-1, 0)
        if rows != batch or page_table.dtype is not _int32_dtype or page_table.device != device:
            _on(page_table, "page_table", device)
            raise ValueError(f"page_table must be int32 [{batch}, max_pages], got {page_table.dtype} {list(page_table.shape)}")
        if not page_table.is_contiguous():
            if page_table.stride(1) != 1 and max_pages > 1:
                raise ValueError("page_table must be contiguous in its last dimension")
            table_stride = page_table.stride(0) if batch > 1 else 0
            if batch > 1 and table_stride < max_pages:  # rows that overlap, an expanded table among them
                raise ValueError("page_table rows must not overlap")
        table = page_table.data_ptr()
    return (k_pages.data_ptr(), v_pages.data_ptr(), kind, pages, hkv, page_size, dim,
            *(_NO_STRIDES[3] if k_pages.is_contiguous() else _strides(k_pages, "k_pages")),
            *(_NO_STRIDES[3] if v_pages.is_contiguous() else _strides(v_pages, "v_pages")),
            0 if k_scale is None else _scale_ptr(k_scale, "k_scale", device, hkv),
            0 if v_scale is None else _scale_ptr(v_scale, "v_scale", device, hkv), table, table_stride, max_pages)


_cache_kinds = _int32_dtype = None


def _cache_kind(dtype):
    global _cache_kinds, _int32_dtype
    if _cache_kinds is None:
        import torch

        _cache_kinds = {torch.bfloat16: ODF_DTYPE_BF16, torch.float8_e4m3fn: ODF_DTYPE_E4M3}
        _int32_dtype = torch.int32
    return _cache_kinds.get(dtype)


def _bad_cache(k_pages, v_pages, device):
    for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages")):
        if t.device != device:
            return ValueError(f"{name} is on {t.device}, the call runs on {device}")
    if k_pages.dtype != v_pages.dtype or _cache_kind(k_pages.dtype) is None:
        return ValueError(f"a cache holds bfloat16 or float8_e4m3fn, not {k_pages.dtype} and {v_pages.dtype}")
    return ValueError("k_pages and v_pages must be rank 4 [pages, heads_kv, page_size, head_dim] of one shape")


class _StayHere:
    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_STAY_HERE = _StayHere()


class _SwitchTo:
    """Makes a device and a stream current, so that what is allocated inside belongs to that stream."""

    def __init__(self, device, handle):
        import torch

        self.device = torch.cuda.device(device)
        self.stream = torch.cuda.stream(torch.cuda.ExternalStream(handle, device=device) if handle
                                        else torch.cuda.default_stream(device))

    def __enter__(self):
        self.device.__enter__()
        self.stream.__enter__()

    def __exit__(self, *exc):
        self.stream.__exit__(*exc)
        return self.device.__exit__(*exc)


def _launch_on(device, stream):
    """(context, stream handle) for a launch on `device` and `stream` (a handle, a torch stream or None
    for torch's current one)."""
    import torch

    # the raw forms of torch.cuda.current_stream(device).cuda_stream and current_device(), which cost 4 us more
    current = torch._C._cuda_getCurrentRawStream(device.index)
    handle = current if stream is None else getattr(stream, "cuda_stream", stream)
    if handle == current and torch._C._cuda_getDevice() == device.index:
        return _STAY_HERE, handle
    return _SwitchTo(device, handle), handle


def _require_cuda(device):
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, not {device}")


def _outputs(q, out, lse_out, out_dtype, want_lse, *lead):
    """The given or new outputs of an attention call with q's shape [*lead, D], and out's dtype code."""
    import torch

    if out is None:
        dtype = out_dtype or torch.float32
        # the short forms of torch.empty(q.shape, dtype=..., device=...), which costs 1 us more
        out = torch.empty_like(q, dtype=dtype) if q.is_contiguous() else q.new_empty(q.shape, dtype=dtype)
    else:
        dtype = out.dtype
        if out.shape != q.shape:
            raise ValueError("out must have q's shape")
        _on(out, "out", q.device)
    if dtype is not torch.bfloat16 and dtype is not torch.float32:
        raise ValueError("out must be float32 or bfloat16")
    code = ODF_DTYPE_BF16 if dtype is torch.bfloat16 else ODF_DTYPE_F32
    if lse_out is None:
        return out, q.new_empty(*lead, dtype=torch.float32) if want_lse else None, code
    _on(lse_out, "lse_out", q.device)
    if lse_out.shape != lead or lse_out.dtype != torch.float32 or not lse_out.is_contiguous():
        raise ValueError("lse_out must be contiguous float32 of q's shape without its last dimension")
    return out, lse_out, code


def _clip(n):
    """A count (or a sequence of a pool) as the C side takes it, where an integer past 64 bits would wrap: below zero
    it is refused there, and past 63 bits no count changes and no sequence is found."""
    return max(-1, min(n, _INT64_MAX))


def _slopes_array(alibi_slopes, heads):
    if alibi_slopes is None:
        return None
    if len(alibi_slopes) != heads:
        raise ValueError("alibi_slopes needs one slope per query head")
    return (C.c_float * heads)(*[float(x) for x in alibi_slopes])


def paged_decode_workspace(batch, heads_q, heads_kv, head_dim, device="cuda"):
    """Scratch for ``paged_decode``, zeroed: a serving loop keeps one per stream for all of its calls."""
    import torch

    p = DecodeParams()
    p.batch, p.heads_q, p.cache.heads_kv, p.cache.head_dim = batch, heads_q, heads_kv, head_dim
    return torch.zeros(load_library().odf_paged_decode_workspace_size(C.byref(p)), dtype=torch.uint8, device=device)


def paged_decode(q, k_pages, v_pages, page_table, lens, *, scale=None, window=0, sinks=0, alibi=False,
                 alibi_slopes=None, softcap=0.0, k_scale=None, v_scale=None, out_dtype=None, want_lse=True, out=None,
                 lse_out=None, workspace=None, stream=None):
    """Attention of one new token per sequence over a paged cache (odf_paged_decode_sm100).

    q [B,Hq,D] bf16; k_pages, v_pages [pages,Hkv,page_size,D] bf16 or float8_e4m3fn (any strides that are
    multiples of 16 bytes, so a [pages,page_size,Hkv,D] cache goes in as a ``transpose(1, 2)`` view);
    page_table int32 [B,max_pages]; lens int32 [B], keys per sequence with the new token's own (append
    first).  ``window`` > 0 keeps the last ``window`` keys and the first ``sinks``.  ``workspace``:
    ``paged_decode_workspace(...)``, kept between calls on one stream; without one, each call makes its own.

    Returns (o [B,Hq,D], lse [B,Hq] fp32 natural log, or None), asynchronous on ``stream``
    (default: torch's current stream).
    """
    import torch

    if q.dim() != 3 or q.dtype != torch.bfloat16:
        raise ValueError("q must be bfloat16 of rank 3 [B, Hq, D]")
    B, Hq, D = q.shape
    dev = q.device
    _require_cuda(dev)
    cache = _cache_params(k_pages, v_pages, k_scale, v_scale, page_table, dev, B, head_dim=D)
    lens_ptr = _int32(lens, "lens", dev, B)
    slopes = _slopes_array(alibi_slopes, Hq) if alibi else None
    where, handle = _launch_on(dev, stream)
    with where:
        out, lse, o_code = _outputs(q, out, lse_out, out_dtype, want_lse, B, Hq)
        if workspace is None:
            workspace = paged_decode_workspace(B, Hq, cache[4], D, device=dev)
        else:
            _on(workspace, "workspace", dev)
        p = _PACK_DECODE(q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                         o_code, B, Hq, *(_NO_STRIDES[2] if q.is_contiguous() else _strides(q, "q")),
                         *(_NO_STRIDES[2] if out.is_contiguous() else _strides(out, "out")), lens_ptr, *cache,
                         1.0 / math.sqrt(D) if scale is None else scale,
                         _clip(window), _clip(sinks), ODF_BIAS_ALIBI if alibi else ODF_BIAS_NONE,
                         0 if slopes is None else C.addressof(slopes), softcap, workspace.data_ptr(), workspace.nbytes)
        _check(load_library().odf_paged_decode_sm100(p, handle))
    return out, (lse if want_lse else None)


def paged_append(k, v, k_pages, v_pages, page_table, starts, *, counts=None, k_scale=None, v_scale=None, stream=None):
    """Writes k, v [B,Hkv,T,D] (bf16) into the cache at positions starts[b] .. (odf_paged_append_sm100).

    Token t of sequence b is written when t < counts[b] (always without ``counts``, int32 [B]).  A
    float8_e4m3fn cache gets x / scale, rounded to nearest and saturated.  Asynchronous on ``stream``.
    """
    import torch

    if k.dim() != 4 or k.shape != v.shape or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("k and v must be bfloat16 of one rank 4 shape [B, Hkv, T, D]")
    B, Hkv, T, D = k.shape
    dev = k.device
    _require_cuda(dev)
    _on(v, "v", dev)
    cache = _cache_params(k_pages, v_pages, k_scale, v_scale, page_table, dev, B, Hkv, D)
    p = _PACK_APPEND(k.data_ptr(), v.data_ptr(), B, T, *_strides(k, "k"), *_strides(v, "v"), _int32(starts, "starts", dev, B),
                     0 if counts is None else _int32(counts, "counts", dev, B), *cache)
    where, handle = _launch_on(dev, stream)
    with where:
        _check(load_library().odf_paged_append_sm100(p, handle))


def _page_ids(pairs, n, pages):
    """The ids of n pairs as an int32 array (and its address), checked before they are cut to 32 bits."""
    if n <= 32:  # a few: plain Python is 3 us faster than numpy
        rows = pairs.tolist() if hasattr(pairs, "tolist") else pairs
        try:
            flat = [operator.index(i) for src, dst in rows for i in (src, dst)]
        except (TypeError, ValueError):
            raise ValueError("pairs must be integers of shape [n, 2]") from None
        if min(flat) < 0 or max(flat) >= pages:
            raise ValueError("a page id is outside the cache")
        ids = (C.c_int32 * (2 * n))(*flat)
        return ids, C.addressof(ids)
    import numpy as np

    ids = np.asarray(pairs)
    if ids.ndim != 2 or ids.shape[1] != 2 or ids.dtype.kind not in "iu":
        raise ValueError("pairs must be integers of shape [n, 2]")
    if ids.dtype != np.int32:
        ids = np.ascontiguousarray(ids, dtype=np.int64)
        if ids.view(np.uint64).max() >= pages:  # negative ids are large here
            raise ValueError("a page id is outside the cache")
    ids = np.ascontiguousarray(ids, dtype=np.int32)
    return ids, ids.ctypes.data


def page_copy(k_pages, v_pages, pairs, *, stream=None):
    """Copies pages pairs[i] = (source, destination) of K and V (odf_page_copy_sm100).

    k_pages, v_pages: one layer [pages,Hkv,page_size,D], or every layer [layers,pages,Hkv,page_size,D] in one
    launch.  ``pairs``: a sequence of pairs, a numpy array or a CPU tensor [n,2], such as
    ``PagePool`` gives out.  Asynchronous on ``stream``.
    """
    rank, shape, dev = k_pages.dim(), k_pages.shape, k_pages.device
    if rank not in (4, 5) or v_pages.shape != shape:
        raise ValueError("k_pages and v_pages must be [pages, Hkv, page_size, D] or [layers, pages, ...] of one shape")
    _require_cuda(dev)
    n = len(pairs)
    if n == 0:
        return
    ids, address = _page_ids(pairs, n, shape[-4])
    cache = _cache_params(k_pages, v_pages, None, None, None, dev, 0)
    layers, k_layer, v_layer = 1, 0, 0
    if rank == 5:
        layers, k_layer, v_layer = shape[0], k_pages.stride(0), v_pages.stride(0)
        if layers == 0:
            raise ValueError("the cache has no layers")
    p = _PACK_COPY(*cache, layers, k_layer, v_layer, address, n)
    where, handle = _launch_on(dev, stream)
    with where:
        _check(load_library().odf_page_copy_sm100(p, handle))
    del ids  # held until the call has read them


class PagePool:
    """Which pages of a cache are free, and every sequence's table (odf_page_pool_*; host only).

    ``extend`` and ``compact`` return (source, destination) pairs for ``page_copy``, to be run before the
    cache is written.  Pairs of consecutive calls of ``extend`` may go into one copy, which has to run before any
    other call that changes the pool (``fork``, ``truncate``, ``free``, ``compact``).  Not thread-safe.
    """

    def __init__(self, num_pages: int, page_size: int):
        self._lib = load_library()
        self._pool = C.c_void_p()
        _check(self._lib.odf_page_pool_create(_clip(num_pages), _clip(page_size), C.byref(self._pool)))
        self.num_pages, self.page_size = num_pages, page_size

    def __del__(self):
        if getattr(self, "_pool", None):
            self._lib.odf_page_pool_destroy(self._pool)
            self._pool = None

    def add(self) -> int:
        """A new, empty sequence."""
        seq = C.c_int64()
        _check(self._lib.odf_page_pool_add(self._pool, C.byref(seq)))
        return seq.value

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens; every page is shared until one of the two writes it."""
        child = C.c_int64()
        _check(self._lib.odf_page_pool_fork(self._pool, _clip(seq), C.byref(child)))
        return child.value

    def extend(self, seq: int, tokens: int) -> list[tuple[int, int]]:
        """Room for ``tokens`` more tokens; raises OdfError(ODF_ERR_NO_PAGES), changing nothing, without it."""
        pair, n = (C.c_int32 * 2)(), C.c_int64()
        _check(self._lib.odf_page_pool_extend(self._pool, _clip(seq), _clip(tokens), pair, C.byref(n)))
        return [(pair[0], pair[1])] if n.value else []

    def truncate(self, seq: int, length: int) -> None:
        """Drops the tokens past ``length``."""
        _check(self._lib.odf_page_pool_truncate(self._pool, _clip(seq), _clip(length)))

    def free(self, seq: int) -> None:
        """Ends a sequence."""
        _check(self._lib.odf_page_pool_free(self._pool, _clip(seq)))

    def compact(self) -> list[tuple[int, int]]:
        """Moves pages so that the used ones are the first ones."""
        room = self.num_pages // 2
        pairs, n = (C.c_int32 * (2 * max(room, 1)))(), C.c_int64()
        _check(self._lib.odf_page_pool_compact(self._pool, pairs, room, C.byref(n)))
        return [(pairs[2 * i], pairs[2 * i + 1]) for i in range(n.value)]

    def length(self, seq: int) -> int:
        tokens, pages = C.c_int64(), C.c_int64()
        _check(self._lib.odf_page_pool_length(self._pool, _clip(seq), C.byref(tokens), C.byref(pages)))
        return tokens.value

    def pages(self, seq: int) -> list[int]:
        tokens, pages = C.c_int64(), C.c_int64()
        _check(self._lib.odf_page_pool_length(self._pool, _clip(seq), C.byref(tokens), C.byref(pages)))
        ids = (C.c_int32 * max(pages.value, 1))()
        _check(self._lib.odf_page_pool_table(self._pool, _clip(seq), ids, pages.value))
        return list(ids[:pages.value])

    def table(self, seqs, max_pages: int | None = None):
        """The page table of a batch: int32 CPU tensor [len(seqs), max_pages], -1 past each sequence's pages."""
        import torch

        rows = [self.pages(s) for s in seqs]
        width = max([1] + [len(r) for r in rows]) if max_pages is None else max_pages
        out = torch.full((len(rows), width), -1, dtype=torch.int32)
        for i, r in enumerate(rows):
            if len(r) > width:
                raise ValueError("a sequence has more pages than the table has entries")
            out[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        return out

    @property
    def free_pages(self) -> int:
        return self._lib.odf_page_pool_free_pages(self._pool)


def device_status(clear=True) -> int:
    v = C.c_int32(0)
    _check(load_library().odf_device_status(C.byref(v), int(clear)))
    return v.value


def env_threads() -> int:
    return max(1, min(os.cpu_count() or 1, 64))
