"""
WidePagedCache: the keys and values of many sequences of N models, in pages of one pool.

    cache.write(k, v, block_table, start, count)      new tokens into the pages
    cache.read(block_table, lengths, max_length)      back to dense [N, B, max_length, Hkv, Dh]
    cache.attend(q, block_table, lengths)             one new token of every sequence over its pages

Token i of sequence (n, b) stands in slot i % page_size of page block_table[n, b, i // page_size] of
the pool (int32 [N, B, M]; entries behind a sequence's last page are not followed and may hold
anything, -1 for example).  Which page is whose is the caller's: pages may be handed out in any
order, and a prefix that several sequences read may be one set of pages.  No two rows of one write
may go to the same slot.  Pools stand as

    k_pages, v_pages     [P, Hkv, page_size, row]      row: head_dim, and zeros up to whole 16 bytes
    k_scales, v_scales   [P, Hkv, page_size]           8-bit caches only

With ``quantized=True`` a row (one head of one token) is 8-bit codes and one fp32 scale: scale =
max(max |x| / 127, 2^-126), code = x / scale to the nearest, ties to even; a row with an infinity
or NaN reads back as NaN.  ``attend`` sums a score before the key's scale multiplies it and takes a
weight times the value's scale as bf16 numbers: queries from 2^110 on can overflow over 8 bits, and
values whose row's largest is under 2^-90 lose bits.

A block-table entry outside the pool, a token past the table's end or a count or length beyond the
call's is never followed: nothing is written there, it reads as zeros, takes no part in the
attention and raises a device-side flag, which ``index_error()`` (synchronises) turns into an
IndexError.  Nothing here allocates pages or advances lengths, and every call reads its tables on
the GPU, so a captured graph replays with whatever they hold then.  The reference has no counterpart.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from .. import _hip, _serve


class WidePagedCache:
    def __init__(self, num_pages: int, page_size: int, n_kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, quantized: bool = False,
                 device: Union[str, torch.device] = "cuda"):
        _hip.dtype_code(dtype, "WidePagedCache")
        stored = torch.int8 if quantized else dtype
        es = torch.empty((), dtype=stored).element_size()
        row = -(-head_dim * es // 16) * 16 // es
        shape = (num_pages, n_kv_heads, page_size)
        pages = lambda: torch.zeros((*shape, row), dtype=stored, device=device)     # noqa: E731
        scales = lambda: torch.zeros(shape, dtype=torch.float32, device=device) if quantized else None  # noqa: E731
        self._adopt(pages(), pages(), scales(), scales(), head_dim, dtype)

    @classmethod
    def from_pages(cls, k_pages: Tensor, v_pages: Tensor, k_scales: Optional[Tensor] = None,
                   v_scales: Optional[Tensor] = None, head_dim: Optional[int] = None,
                   dtype: Optional[torch.dtype] = None) -> "WidePagedCache":
        """A cache over pools that exist (not copied): int8 pages with their scales, of a cache for ``dtype``, or pages
        of a floating dtype.  Rows are whole 16 bytes; columns from ``head_dim`` on hold zeros."""
        self = cls.__new__(cls)
        self._adopt(k_pages, v_pages, k_scales, v_scales, k_pages.shape[-1] if head_dim is None else head_dim,
                    k_pages.dtype if dtype is None else dtype)
        return self

    def _adopt(self, k_pages, v_pages, k_scales, v_scales, head_dim, dtype) -> None:
        what = "WidePagedCache"
        code = _hip.dtype_code(dtype, what)
        quantized = k_pages.dtype == torch.int8
        _hip.require_device(what, k_pages, v_pages, k_scales, v_scales)
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype:
            raise ValueError(f"{what}: k and v pages must be two [P, Hkv, page_size, row] tensors of one dtype")
        if not quantized and k_pages.dtype != dtype:
            raise ValueError(f"{what}: pages of {k_pages.dtype} in a cache for {dtype}")
        pages, heads, page_size, row = k_pages.shape
        if (k_scales is None) == quantized or (v_scales is None) == quantized:
            raise ValueError(f"{what}: 8-bit pages, and only they, come with k and v scales")
        for t in (k_scales, v_scales):
            if t is not None and (t.dtype != torch.float32 or t.shape != k_pages.shape[:3]):
                raise ValueError(f"{what}: scales must be float32 [P, Hkv, page_size]")
        if not all(t is None or t.is_contiguous() for t in (k_pages, v_pages, k_scales, v_scales)):
            raise ValueError(f"{what}: pools must be contiguous")
        _serve.same_device(what, k_pages, v_pages, k_scales, v_scales)
        if not 0 < head_dim <= min(row, 256):
            raise ValueError(f"{what}: head_dim {head_dim} must be within [1, {min(row, 256)}]")
        if heads < 1:
            raise ValueError(f"{what}: n_kv_heads must be positive")
        if page_size < 1 or row * k_pages.element_size() % 16 or row > 512:
            raise ValueError(f"{what}: pages of at least one token, rows of whole 16 bytes and at most 512 elements, "
                             f"got {page_size} and {row}")
        self._pools = (k_pages, v_pages, k_scales, v_scales)
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = pages, heads, page_size, head_dim
        self.dtype, self.quantized, self.device = dtype, quantized, k_pages.device
        self._err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._sizes = (code, 8 if quantized else 0, pages, page_size, heads, head_dim, row)
        self._plans = _serve.Plans()

    def _sizes_for(self, n: int, b: int) -> Tuple:
        return (*self._sizes[:2], n, b, *self._sizes[2:])

    # The pools are this cache's for good: its plans hold their sizes.
    @property
    def k_pages(self) -> Tensor:
        return self._pools[0]

    @property
    def v_pages(self) -> Tensor:
        return self._pools[1]

    @property
    def k_scales(self) -> Optional[Tensor]:
        return self._pools[2]

    @property
    def v_scales(self) -> Optional[Tensor]:
        return self._pools[3]

    @staticmethod
    def _check_table(what: str, table: Tensor, n: int, b: int) -> None:
        if table.dim() != 3 or table.dtype != torch.int32 or table.shape[0] != n or table.shape[1] != b:
            raise RuntimeError(f"{what}: block_table must be int32 [N={n}, B={b}, M], got {table.dtype} {list(table.shape)}")

    @staticmethod
    def _check_per_sequence(what: str, name: str, t: Optional[Tensor], n: int, b: int) -> None:
        if t is not None and (t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != n or t.shape[1] != b):
            raise RuntimeError(f"{what}: {name} must be int32 [N={n}, B={b}], got {t.dtype} {list(t.shape)}")

    @staticmethod
    def _dense(t: Optional[Tensor]) -> Optional[Tensor]:
        return t if t is None or t.is_contiguous() else t.contiguous()

    def write(self, k: Tensor, v: Tensor, block_table: Tensor, start: Tensor, count: Optional[Tensor] = None) -> None:
        """Rows [0, count[n, b]) of k, v [N, B, T, Hkv, Dh] become tokens start[n, b] + 0, 1, ... of their
        sequences (count None: all T).  Rows from count on are padding, and a sequence of negative start takes part in
        nothing: neither is written."""
        if torch.compiler.is_compiling():
            return _serve.uncompiled(self.write, k, v, block_table, start, count)
        form = (k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype, v.get_device(),
                block_table.shape, block_table.dtype, block_table.get_device(), start.shape, start.dtype, start.get_device(),
                None if count is None else (count.shape, count.dtype, count.get_device()))
        plan = self._plans.get(form)
        if plan is None:
            what = "WidePagedCache.write"
            _hip.require_device(what, k, v, block_table, start, count)
            if k.dim() != 5 or k.shape != v.shape or k.shape[3] != self.n_kv_heads or k.shape[4] != self.head_dim:
                raise RuntimeError(f"{what}: k and v must be [N, B, T, {self.n_kv_heads}, {self.head_dim}], got "
                                   f"{list(k.shape)} and {list(v.shape)}")
            if k.dtype != self.dtype or v.dtype != self.dtype:
                raise RuntimeError(f"{what}: k {k.dtype} and v {v.dtype} in a cache for {self.dtype}")
            n, b = k.shape[:2]
            self._check_table(what, block_table, n, b)
            self._check_per_sequence(what, "start", start, n, b)
            self._check_per_sequence(what, "count", count, n, b)
            _serve.same_device(what, self.k_pages, k, v, block_table, start, count)
            plan = self._plans.keep(form, self._sizes_for(n, b))
        if torch.is_grad_enabled():
            _hip.require_forward_only("WidePagedCache.write", k, v)
        k = k if k.stride(4) == 1 else k.contiguous()
        v = v if v.stride(4) == 1 else v.contiguous()
        _serve.cache_write(self, plan, k, v, self._dense(block_table), self._dense(start), self._dense(count))

    def read(self, block_table: Tensor, lengths: Tensor, max_length: int) -> Tuple[Tensor, Tensor]:
        """K and V of tokens [0, lengths[n, b]) as [N, B, max_length, Hkv, Dh]; zeros from a sequence's length on."""
        if torch.compiler.is_compiling():
            return _serve.uncompiled(self.read, block_table, lengths, max_length)
        form = (block_table.shape, block_table.dtype, block_table.get_device(), lengths.shape, lengths.dtype,
                lengths.get_device())
        sizes = self._plans.get(form)
        if max_length < 0:
            raise RuntimeError(f"WidePagedCache.read: max_length must not be negative, got {max_length}")
        if sizes is None:
            what = "WidePagedCache.read"
            _hip.require_device(what, block_table, lengths)
            n, b = block_table.shape[:2]
            self._check_table(what, block_table, n, b)
            self._check_per_sequence(what, "lengths", lengths, n, b)
            _serve.same_device(what, self.k_pages, block_table, lengths)
            sizes = self._plans.keep(form, self._sizes_for(n, b))
        shape = (*lengths.shape, max_length, self.n_kv_heads, self.head_dim)
        k = torch.empty(shape, dtype=self.dtype, device=self.device)
        v = torch.empty(shape, dtype=self.dtype, device=self.device)
        if k.numel():
            _serve.cache_read(self, sizes, self._dense(block_table), self._dense(lengths), max_length, k, v)
        return k, v

    def attend(self, q: Tensor, block_table: Tensor, lengths: Tensor, first: Optional[Tensor] = None,
               scale: Optional[float] = None, max_length: Optional[int] = None) -> Tensor:
        """softmax(scale q k^T) v of one new token per sequence, q [N, B, Hq, Dh], over cached tokens
        [first[n, b], lengths[n, b]) (first None: from 0; a window of w tokens is first = lengths - w).  Query
        head h reads key head h // (Hq // Hkv); scale defaults to Dh ** -0.5.  A sequence without tokens gets
        zeros.  ``max_length`` bounds the lengths (default: what the block table can name); a tight bound splits
        short sequences less."""
        if torch.compiler.is_compiling():
            return _serve.uncompiled(self.attend, q, block_table, lengths, first, scale, max_length)
        form = (q.shape, q.dtype, q.get_device(), block_table.shape, block_table.dtype, block_table.get_device(),
                lengths.shape, lengths.dtype, lengths.get_device(),
                None if first is None else (first.shape, first.dtype, first.get_device()))
        plan = self._plans.get(form)
        if plan is None:
            plan = self._plans.keep(form, self._plan_attend(q, block_table, lengths, first))
        sizes, reach, needs = plan
        most = reach if max_length is None else max_length
        need = needs.get(most)
        if need is None:
            need = needs.keep(most, self._workspace(sizes, q, block_table, most))
        if torch.is_grad_enabled():
            _hip.require_forward_only("WidePagedCache.attend", q)
        q = q if q.stride(3) == 1 else q.contiguous()
        o = q.new_empty(q.shape)
        if o.numel():
            ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            _serve.paged_attention(self, sizes, q, o, self._dense(block_table), self._dense(lengths), self._dense(first),
                                   self.head_dim ** -0.5 if scale is None else scale, most, ws)
        return o

    def _plan_attend(self, q: Tensor, block_table: Tensor, lengths: Tensor, first: Optional[Tensor]) -> Tuple:
        what = "WidePagedCache.attend"
        _hip.require_device(what, q, block_table, lengths, first)
        if q.dim() != 4 or q.shape[3] != self.head_dim or q.shape[2] % self.n_kv_heads:
            raise RuntimeError(f"{what}: q must be [N, B, a multiple of {self.n_kv_heads} heads, {self.head_dim}], got "
                               f"{list(q.shape)}")
        if q.dtype != self.dtype:
            raise RuntimeError(f"{what}: q {q.dtype} over a cache for {self.dtype}")
        n, b = q.shape[:2]
        self._check_table(what, block_table, n, b)
        self._check_per_sequence(what, "lengths", lengths, n, b)
        self._check_per_sequence(what, "first", first, n, b)
        _serve.same_device(what, self.k_pages, q, block_table, lengths, first)
        # workspaces by max_length, which a caller may raise with every token: apart from the checks above
        return self._sizes_for(n, b), min(block_table.shape[2] * self.page_size, 2 ** 31 - 65), _serve.Plans()

    def _workspace(self, sizes: Tuple, q: Tensor, block_table: Tensor, max_length: int) -> int:
        if max_length < 0:
            raise RuntimeError(f"WidePagedCache.attend: max_length must not be negative, got {max_length}")
        return _serve.paged_attention_workspace(self, sizes, block_table, q.shape[2], max_length) if q.numel() else 0

    def index_error(self) -> None:
        """Raise IndexError if any call since the last check met a page outside the pool, or a token, count or length
        past its bounds."""
        if int(self._err.item()) != 0:
            self._err.zero_()
            raise IndexError("WidePagedCache: a block-table entry, token, count or length was out of range")

    def __repr__(self) -> str:
        return (f"WidePagedCache({self.num_pages} pages of {self.page_size}, heads={self.n_kv_heads}, "
                f"head_dim={self.head_dim}, {'int8 for ' if self.quantized else ''}{self.dtype})")


__all__ = ["WidePagedCache"]
