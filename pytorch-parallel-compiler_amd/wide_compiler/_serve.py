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


# Plans: what a call's sizes, strides and types come to, worked out (and checked) once for each form of a call and
# kept by the module or cache that is called: the leading fields of the argument struct.  The tensors' addresses are
# read on every call.

class Plans(dict):
    """Plans by the form of a call; a program that never repeats a form does not fill memory with them."""

    def keep(self, form, plan):
        if len(self) >= 256:
            self.clear()
        self[form] = plan
        return plan


def head_norm_plan(*, q: Tensor, k: Tensor, q_weight: Tensor, positions: Tensor, rotary_dim: int,
                   interleaved: bool) -> Tuple:
    """q [N, B, T, Hq, Dh], k [N, B, T, Hk, Dh] (unit last stride), positions expanded to [N, B, T]."""
    n, b, t, hq, dh = q.shape
    return ((_hip.dtype_code(q.dtype, "head_norm"), _hip.dtype_code(q_weight.dtype, "head_norm"),
             1 if interleaved else 0, positions.element_size(), n, b, t, hq, k.shape[3], dh, rotary_dim),
            q.stride()[:4], k.stride()[:4], positions.stride())


def head_norm_rotary(plan, q: Tensor, k: Tensor, q_out: Tensor, k_out: Tensor, q_weight: Tensor, k_weight: Tensor,
                     freq: Tensor, positions: Tensor, eps: float) -> None:
    """q_out, k_out contiguous; freq the turns per position as the bits of fp64."""
    sizes, q_strides, k_strides, p_strides = plan
    _launch("wc_head_norm_rotary", _HeadNormArgs, _pack_head_norm(
        *sizes, q.data_ptr(), *q_strides, k.data_ptr(), *k_strides, q_out.data_ptr(), k_out.data_ptr(),
        q_weight.data_ptr(), k_weight.data_ptr(), freq.data_ptr(), positions.data_ptr(), *p_strides, eps), q)


def _cache_fields(cache, sizes: Tuple, table: Tensor) -> Tuple:
    k, v, ks, vs = cache._pools
    m = table.shape[2]
    return (*sizes, k.data_ptr(), v.data_ptr(), 0 if ks is None else ks.data_ptr(), 0 if vs is None else vs.data_ptr(),
            table.data_ptr(), m, m, cache._err.data_ptr())


def cache_write(cache, sizes: Tuple, k: Tensor, v: Tensor, table: Tensor, start: Tensor,
                count: Optional[Tensor]) -> None:
    _launch("wc_cache_write", _CacheWriteArgs, _pack_write(
        *_cache_fields(cache, sizes, table), k.shape[2], k.data_ptr(), *k.stride()[:4], v.data_ptr(), *v.stride()[:4],
        start.data_ptr(), 0 if count is None else count.data_ptr()), k)


def cache_read(cache, sizes: Tuple, table: Tensor, lengths: Tensor, max_length: int, k: Tensor, v: Tensor) -> None:
    _launch("wc_cache_read", _CacheReadArgs, _pack_read(
        *_cache_fields(cache, sizes, table), lengths.data_ptr(), max_length, k.data_ptr(), v.data_ptr()), table)


def paged_attention_workspace(cache, sizes: Tuple, table: Tensor, heads: int, max_length: int) -> int:
    """Bytes of workspace that attention of `heads` query heads takes."""
    a = _PagedAttnArgs.from_buffer_copy(_pack_attn(*_cache_fields(cache, sizes, table), heads, max_length, 0, 0, 0, 0,
                                                   0, 0, 0, 0, 0, 0.0))
    need = int(lib().wc_paged_attention_workspace_bytes(ctypes.byref(a)))
    if need < 0:
        raise _hip.WideKernelError(f"wc_paged_attention: {_hip.last_error()}")
    return need


def paged_attention(cache, sizes: Tuple, q: Tensor, o: Tensor, table: Tensor, lengths: Tensor, first: Optional[Tensor],
                    scale: float, max_length: int, workspace: Optional[Tensor]) -> None:
    _launch("wc_paged_attention", _PagedAttnArgs, _pack_attn(
        *_cache_fields(cache, sizes, table), q.shape[2], max_length, q.data_ptr(), *q.stride()[:3], o.data_ptr(),
        lengths.data_ptr(), 0 if first is None else first.data_ptr(),
        *((0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())), scale), q)


def linear4(sizes: Tuple, rows, x: Tensor, codes: Tensor, scales: Tensor, zeros: Tensor, bias: Optional[Tensor],
            y: Tensor) -> None:
    """sizes: dtype, group, n, m, o, k; rows the strides of x (_layout.Rows)."""
    _launch("wc_linear4", _Linear4Args, _pack_linear4(
        *sizes, x.data_ptr(), rows[0], rows[1], rows[2], rows[3], codes.data_ptr(), scales.data_ptr(), zeros.data_ptr(),
        0 if bias is None else bias.data_ptr(), y.data_ptr()), x)


@torch.compiler.disable
def uncompiled(call, *args):
    """call(*args) outside a region that torch.compile traces: what the modules' and the cache's calls do there, whose
    plans and launches are nothing to trace.  A check of is_compiling() costs a call less than the decorator does.  An
    export has no outside: it would come back here for ever."""
    if torch.compiler.is_compiling():
        raise RuntimeError(f"{getattr(call, '__qualname__', call)}: a kernel's launch cannot be exported")
    return call(*args)
