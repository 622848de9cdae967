"""
Binding of the decode-step kernels of libwide_hip.so (include/wc_serve_abi.h): head norms with
rotation, the paged key-value cache, attention of one new token over it, products with 4-bit
weights.  Like _hip, thin wrappers that fill an argument struct and launch on torch's current
stream; the modules that call them check the tensors.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _hip

ABI_VERSION = 1

_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class _HeadNormArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", _I32), ("param_dtype", _I32), ("interleaved", _I32), ("position_bytes", _I32),
        ("n", _I64), ("b", _I64), ("t", _I64), ("q_heads", _I64), ("k_heads", _I64),
        ("head_dim", _I64), ("rotary_dim", _I64),
        ("q", _P), ("q_stride_n", _I64), ("q_stride_b", _I64), ("q_stride_t", _I64), ("q_stride_h", _I64),
        ("k", _P), ("k_stride_n", _I64), ("k_stride_b", _I64), ("k_stride_t", _I64), ("k_stride_h", _I64),
        ("q_out", _P), ("k_out", _P), ("q_weight", _P), ("k_weight", _P), ("freq", _P), ("positions", _P),
        ("p_stride_n", _I64), ("p_stride_b", _I64), ("p_stride_t", _I64), ("eps", _F),
    ]


class _PagedCache(ctypes.Structure):
    _fields_ = [
        ("dtype", _I32), ("bits", _I32), ("n", _I64), ("b", _I64),
        ("pages", _I64), ("page_size", _I64), ("heads", _I64), ("head_dim", _I64), ("row", _I64),
        ("k_pages", _P), ("v_pages", _P), ("k_scales", _P), ("v_scales", _P),
        ("table", _P), ("table_len", _I64), ("table_stride", _I64), ("err_flag", _P),
    ]


class _CacheWriteArgs(ctypes.Structure):
    _fields_ = [
        *_PagedCache._fields_, ("t", _I64),              # the embedded wc_paged_cache first
        ("k", _P), ("k_stride_n", _I64), ("k_stride_b", _I64), ("k_stride_t", _I64), ("k_stride_h", _I64),
        ("v", _P), ("v_stride_n", _I64), ("v_stride_b", _I64), ("v_stride_t", _I64), ("v_stride_h", _I64),
        ("start", _P), ("count", _P),
    ]


class _CacheReadArgs(ctypes.Structure):
    _fields_ = [*_PagedCache._fields_, ("lengths", _P), ("max_length", _I64), ("k", _P), ("v", _P)]


class _PagedAttnArgs(ctypes.Structure):
    _fields_ = [
        *_PagedCache._fields_, ("q_heads", _I64), ("max_length", _I64),
        ("q", _P), ("q_stride_n", _I64), ("q_stride_b", _I64), ("q_stride_h", _I64), ("o", _P),
        ("lengths", _P), ("first", _P), ("workspace", _P), ("workspace_bytes", _I64), ("scale", _F),
    ]


class _Linear4Args(ctypes.Structure):
    _fields_ = [
        ("dtype", _I32), ("group", _I32), ("n", _I64), ("m", _I64), ("o", _I64), ("k", _I64),
        ("x", _P), ("x_stride_n", _I64), ("x_stride_outer", _I64), ("x_stride_inner", _I64), ("x_rows_inner", _I64),
        ("codes", _P), ("scales", _P), ("zeros", _P), ("bias", _P), ("y", _P),
    ]


_pack_head_norm, _pack_write, _pack_read, _pack_attn, _pack_linear4 = (
    _hip._packer(c) for c in (_HeadNormArgs, _CacheWriteArgs, _CacheReadArgs, _PagedAttnArgs, _Linear4Args))

# name -> (restype, argtypes): what include/wc_serve_abi.h declares
SIGNATURES = {
    "wc_serve_abi_version": (_I32, []),
    "wc_head_norm_rotary": (_I32, [ctypes.POINTER(_HeadNormArgs), _P]),
    "wc_cache_write": (_I32, [ctypes.POINTER(_CacheWriteArgs), _P]),
    "wc_cache_read": (_I32, [ctypes.POINTER(_CacheReadArgs), _P]),
    "wc_paged_attention_workspace_bytes": (_I64, [ctypes.POINTER(_PagedAttnArgs)]),
    "wc_paged_attention": (_I32, [ctypes.POINTER(_PagedAttnArgs), _P]),
    "wc_linear4": (_I32, [ctypes.POINTER(_Linear4Args), _P]),
}

_lib = None


def lib():
    """libwide_hip.so with the entry points of wc_serve_abi.h declared."""
    global _lib
    if _lib is None:
        handle = _hip.lib()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype, fn.argtypes = res, args
        got = handle.wc_serve_abi_version()
        if got != ABI_VERSION:
            raise ImportError(f"wide_compiler: libwide_hip.so serve ABI {got} != expected {ABI_VERSION}")
        _lib = handle
    return _lib


def _launch(name: str, cls, block: bytes, like: Tensor) -> None:
    """Call `name` on the current stream of like's device, which is the current device for the call."""
    if _lib is None:
        lib()
    if like.get_device() != torch.cuda.current_device():
        with torch.cuda.device(like.device):
            return _hip._launch(name, cls, block, _hip.stream_of(like))
    _hip._launch(name, cls, block, _hip.stream_of(like))


def same_device(what: str, like: Tensor, *tensors: Optional[Tensor]) -> None:
    for t in tensors:
        if t is not None and t.device != like.device:
            raise RuntimeError(f"{what}: tensors on {like.device} and {t.device}; one call takes one device")


def head_norm_rotary(*, q: Tensor, k: Tensor, q_out: Tensor, k_out: Tensor, q_weight: Tensor, k_weight: Tensor,
                     freq: Tensor, positions: Tensor, rotary_dim: int, interleaved: bool, eps: float) -> None:
    """q [N, B, T, Hq, Dh], k [N, B, T, Hk, Dh] (unit last stride), positions expanded to [N, B, T]; q_out, k_out
    contiguous; freq the turns per position as the bits of fp64."""
    n, b, t, hq, dh = q.shape
    _launch("wc_head_norm_rotary", _HeadNormArgs, _pack_head_norm(
        _hip.dtype_code(q.dtype, "head_norm"), _hip.dtype_code(q_weight.dtype, "head_norm"), 1 if interleaved else 0,
        positions.element_size(), n, b, t, hq, k.shape[3], dh, rotary_dim,
        q.data_ptr(), *q.stride()[:4], k.data_ptr(), *k.stride()[:4], q_out.data_ptr(), k_out.data_ptr(),
        q_weight.data_ptr(), k_weight.data_ptr(), freq.data_ptr(), positions.data_ptr(), *positions.stride(), eps), q)


def _cache_fields(cache, table: Tensor, n: int, b: int) -> Tuple:
    return (*cache._sizes[:2], n, b, *cache._sizes[2:], cache.k_pages.data_ptr(), cache.v_pages.data_ptr(),
            0 if cache.k_scales is None else cache.k_scales.data_ptr(),
            0 if cache.v_scales is None else cache.v_scales.data_ptr(),
            table.data_ptr(), table.shape[2], table.shape[2], cache._err.data_ptr())


def cache_write(cache, k: Tensor, v: Tensor, table: Tensor, start: Tensor, count: Optional[Tensor]) -> None:
    n, b, t = k.shape[:3]
    _launch("wc_cache_write", _CacheWriteArgs, _pack_write(
        *_cache_fields(cache, table, n, b), t, k.data_ptr(), *k.stride()[:4], v.data_ptr(), *v.stride()[:4],
        start.data_ptr(), 0 if count is None else count.data_ptr()), k)


def cache_read(cache, table: Tensor, lengths: Tensor, max_length: int, k: Tensor, v: Tensor) -> None:
    n, b = table.shape[:2]
    _launch("wc_cache_read", _CacheReadArgs, _pack_read(
        *_cache_fields(cache, table, n, b), lengths.data_ptr(), max_length, k.data_ptr(), v.data_ptr()), table)


def paged_attention(cache, q: Tensor, o: Tensor, table: Tensor, lengths: Tensor, first: Optional[Tensor],
                    scale: float, max_length: int, workspace_of) -> None:
    """workspace_of(bytes): a workspace tensor; called only where the sizes need one."""
    n, b, heads = q.shape[:3]
    fields = (*_cache_fields(cache, table, n, b), heads, max_length, q.data_ptr(), *q.stride()[:3], o.data_ptr(),
              lengths.data_ptr(), 0 if first is None else first.data_ptr())
    block = _pack_attn(*fields, 0, 0, scale)
    need = int(lib().wc_paged_attention_workspace_bytes(ctypes.byref(_PagedAttnArgs.from_buffer_copy(block))))
    if need < 0:
        raise _hip.WideKernelError(f"wc_paged_attention: {_hip.last_error()}")
    ws = None
    if need:
        ws = workspace_of(need)
        block = _pack_attn(*fields, ws.data_ptr(), need, scale)
    _launch("wc_paged_attention", _PagedAttnArgs, block, q)


def linear4(*, n: int, m: int, o: int, k: int, group: int, x: Tensor, rows, codes: Tensor, scales: Tensor,
            zeros: Tensor, bias: Optional[Tensor], y: Tensor) -> None:
    _launch("wc_linear4", _Linear4Args, _pack_linear4(
        _hip.dtype_code(x.dtype, "linear4"), group, n, m, o, k, x.data_ptr(), rows.stride_n, rows.stride_outer,
        rows.stride_inner, rows.rows_inner, codes.data_ptr(), scales.data_ptr(),
        zeros.data_ptr(), 0 if bias is None else bias.data_ptr(), y.data_ptr()), x)


for _name in ("head_norm_rotary", "cache_write", "cache_read", "paged_attention", "linear4"):
    globals()[_name] = torch.compiler.disable(globals()[_name])
del _name
