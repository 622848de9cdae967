"""
Binding of the kernels of libwide_hip.so that draw many answers to the same prompts (include/wc_answer_abi.h):
attention over a prefix that sequences share, products in 8-bit integers, sampling.  Like _serve, thin wrappers
that fill an argument struct and launch on torch's current stream; the modules that call them check the tensors.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _hip, _serve

ABI_VERSION = 1

_P, _I32, _I64, _F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float


class _SharedAttnArgs(ctypes.Structure):
    _fields_ = [
        *_serve._PagedCache._fields_, ("share", _I64), ("prefix_table", _P), ("prefix_len", _I64), ("prefix_stride", _I64),
        ("prefix_lengths", _P), ("q_heads", _I64), ("max_prefix", _I64), ("max_length", _I64),
        ("q", _P), ("q_stride_n", _I64), ("q_stride_b", _I64), ("q_stride_h", _I64), ("o", _P),
        ("lengths", _P), ("workspace", _P), ("workspace_bytes", _I64), ("scale", _F),
    ]


class _Linear8Args(ctypes.Structure):
    _fields_ = [
        ("dtype", _I32), ("n", _I64), ("m", _I64), ("o", _I64), ("k", _I64),
        ("x", _P), ("x_stride_n", _I64), ("x_stride_outer", _I64), ("x_stride_inner", _I64), ("x_rows_inner", _I64),
        ("codes", _P), ("scales", _P), ("bias", _P), ("y", _P), ("workspace", _P), ("workspace_bytes", _I64),
    ]


class _SampleArgs(ctypes.Structure):
    _fields_ = [
        ("dtype", _I32), ("n", _I64), ("m", _I64), ("v", _I64),
        ("logits", _P), ("x_stride_n", _I64), ("x_stride_outer", _I64), ("x_stride_inner", _I64), ("x_rows_inner", _I64),
        ("u", _P), ("temperature", _P), ("top_k", _P), ("top_p", _P), ("min_p", _P),
        ("temperature_stride_n", _I64), ("temperature_stride_m", _I64), ("top_k_stride_n", _I64), ("top_k_stride_m", _I64),
        ("top_p_stride_n", _I64), ("top_p_stride_m", _I64), ("min_p_stride_n", _I64), ("min_p_stride_m", _I64),
        ("tokens", _P), ("workspace", _P), ("workspace_bytes", _I64),
    ]


_pack_shared, _pack_linear8, _pack_sample = (_hip._packer(c) for c in (_SharedAttnArgs, _Linear8Args, _SampleArgs))

# name -> (restype, argtypes): what include/wc_answer_abi.h declares
SIGNATURES = {
    "wc_answer_abi_version": (_I32, []),
    "wc_shared_attention_workspace_bytes": (_I64, [ctypes.POINTER(_SharedAttnArgs)]),
    "wc_shared_attention": (_I32, [ctypes.POINTER(_SharedAttnArgs), _P]),
    "wc_linear8_workspace_bytes": (_I64, [ctypes.POINTER(_Linear8Args)]),
    "wc_linear8": (_I32, [ctypes.POINTER(_Linear8Args), _P]),
    "wc_sample_workspace_bytes": (_I64, [ctypes.POINTER(_SampleArgs)]),
    "wc_sample": (_I32, [ctypes.POINTER(_SampleArgs), _P]),
}

_lib = None


def lib():
    """libwide_hip.so with the entry points of wc_answer_abi.h declared."""
    global _lib
    if _lib is None:
        handle = _serve.lib()
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype, fn.argtypes = res, args
        got = handle.wc_answer_abi_version()
        if got != ABI_VERSION:
            raise ImportError(f"wide_compiler: libwide_hip.so answer ABI {got} != expected {ABI_VERSION}")
        _lib = handle
    return _lib


def _launch(name: str, cls, block: bytes, like: Tensor) -> None:
    if _lib is None:
        lib()
    _serve._launch(name, cls, block, like)


def _workspace(name: str, cls, block: bytes) -> int:
    """Bytes of workspace that a call of these sizes takes."""
    need = int(getattr(lib(), name + "_workspace_bytes")(ctypes.byref(cls.from_buffer_copy(block))))
    if need < 0:
        raise _hip.WideKernelError(f"{name}: {_hip.last_error()}")
    return need


def workspace(like: Tensor, need: int) -> Tuple[Optional[Tensor], int]:
    """A call's workspace, and its address: one for every call, so that calls on several streams and captured graphs
    share none."""
    if not need:
        return None, 0
    ws = torch.empty(need, dtype=torch.uint8, device=like.device)
    return ws, ws.data_ptr()


def linear8_workspace(sizes: Tuple) -> int:
    """sizes: dtype, n, m, o, k."""
    return _workspace("wc_linear8", _Linear8Args, _pack_linear8(*sizes, *(0,) * 11))


def linear8(sizes: Tuple, rows, need: int, x: Tensor, codes: Tensor, scales: Tensor, bias: Optional[Tensor], y: Tensor) -> None:
    """rows: the strides of x (_layout.Rows); scales: fp32, or their bits."""
    ws, at = workspace(x, need)
    _launch("wc_linear8", _Linear8Args, _pack_linear8(
        *sizes, x.data_ptr(), rows[0], rows[1], rows[2], rows[3], codes.data_ptr(), scales.data_ptr(),
        0 if bias is None else bias.data_ptr(), y.data_ptr(), at, need), x)


def sample_workspace(sizes: Tuple) -> int:
    """sizes: dtype, n, m, v."""
    return _workspace("wc_sample", _SampleArgs, _pack_sample(*sizes, *(0,) * 21))


def sample(sizes: Tuple, rows, need: int, logits: Tensor, u: Tensor, rules, strides: Tuple, tokens: Tensor) -> None:
    """rows: the strides of the logits (_layout.Rows); rules: the addresses of temperature, top_k, top_p and min_p."""
    ws, at = workspace(logits, need)
    _launch("wc_sample", _SampleArgs, _pack_sample(
        *sizes, logits.data_ptr(), rows[0], rows[1], rows[2], rows[3], u.data_ptr(), *rules, *strides, tokens.data_ptr(),
        at, need), logits)


def shared_attention_workspace(sizes: Tuple, table_len: int, share: int, prefix_len: int, heads: int, max_prefix: int,
                               max_length: int) -> int:
    """Bytes of workspace that attention of `heads` query heads takes."""
    return _workspace("wc_shared_attention", _SharedAttnArgs, _pack_shared(
        *sizes, 0, 0, 0, 0, 0, table_len, table_len, 0, share, 0, prefix_len, prefix_len, 0, heads, max_prefix, max_length,
        *(0,) * 8, 0.0))


def shared_attention(cache, sizes: Tuple, share: int, q: Tensor, o: Tensor, prefix_table: Tensor, prefix_lengths: Tensor,
                     table: Tensor, lengths: Tensor, scale: float, most: Tuple[int, int], need: int) -> None:
    ws, at = workspace(q, need)
    m = prefix_table.shape[2]
    _launch("wc_shared_attention", _SharedAttnArgs, _pack_shared(
        *_serve._cache_fields(cache, sizes, table), share, prefix_table.data_ptr(), m, m, prefix_lengths.data_ptr(),
        q.shape[2], *most, q.data_ptr(), *q.stride()[:3], o.data_ptr(), lengths.data_ptr(), at, need, scale), q)
