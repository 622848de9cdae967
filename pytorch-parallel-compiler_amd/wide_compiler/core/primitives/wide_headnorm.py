"""
WideHeadNormRotary: the norms of queries and keys and their rotation by position, of N models.

    forward(q, k, positions)   q [N, B, T, Hq, Dh], k [N, B, T, Hk, Dh]  ->  both, of the same shapes

Every head of every token is divided by its root mean square, multiplied by its model's weight
(q_weight or k_weight, [N, Dh]) and turned: with angle a = position * base^(-2p / rotary_dim),

    (y_a, y_b) -> (y_a cos a - y_b sin a, y_b cos a + y_a sin a)

for the pairs p of the first ``rotary_dim`` columns: columns (p, p + rotary_dim / 2), or
neighbours (2p, 2p + 1) when ``interleaved``.  Angles are taken in 64 bits, so that a token at any
position up to 2^28 turns as exactly as the first (fp32 would be off by a radian at 2^24).  Squares
are summed in fp32, as nn.RMSNorm sums them.  ``positions`` is an integer tensor that broadcasts
to [N, B, T].  q and k may be views (of one projection's output, say) with unit last stride.  One
launch of wc_head_norm_rotary; the reference has no counterpart.
"""

from __future__ import annotations

import math
from typing import List, Optional, Tuple

import torch
from torch import Tensor, nn

from ... import _hip, _serve


class WideHeadNormRotary(nn.Module):
    def __init__(self, n: int, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0,
                 eps: float = 1e-6, interleaved: bool = False):
        super().__init__()
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim % 2 or head_dim > 256:
            raise ValueError(f"WideHeadNormRotary: head_dim must be even and at most 256, got {head_dim}")
        if rotary_dim % 2 or not 0 <= rotary_dim <= head_dim:
            raise ValueError(f"WideHeadNormRotary: rotary_dim must be even and within [0, {head_dim}], got {rotary_dim}")
        self.n = n
        self.head_dim = head_dim
        self._rotation = (rotary_dim, base, interleaved)
        self.eps = eps
        self.q_weight = nn.Parameter(torch.ones(n, head_dim))
        self.k_weight = nn.Parameter(torch.ones(n, head_dim))
        # turns per position, as the bits of fp64: .to(dtype) leaves integer buffers as they are
        self.register_buffer("_freq_bits", self._frequencies(None), persistent=False)
        self._plans = _serve.Plans()

    def _frequencies(self, device: Optional[torch.device]) -> Tensor:
        rotary_dim, base, _ = self._rotation
        turns = [base ** (-2.0 * p / rotary_dim) / (2.0 * math.pi) for p in range(rotary_dim // 2)]
        return torch.tensor(turns, dtype=torch.float64, device=device).view(torch.int64)

    def _apply(self, fn, recurse: bool = True):
        """No state_dict holds the frequencies, and to_empty() leaves a module that was made on the meta device with whatever
        stood in memory: wherever the module goes they are made again."""
        super()._apply(fn, recurse)
        device = self._buffers["_freq_bits"].device
        self._buffers["_freq_bits"] = self._frequencies(device)
        return self

    # What turns the heads is a module's for good: its frequencies and its plans are made of it.
    @property
    def rotary_dim(self) -> int:
        return self._rotation[0]

    @property
    def base(self) -> float:
        return self._rotation[1]

    @property
    def interleaved(self) -> bool:
        return self._rotation[2]

    def forward(self, q: Tensor, k: Tensor, positions: Tensor) -> Tuple[Tensor, Tensor]:
        if torch.compiler.is_compiling():
            return _serve.uncompiled(self.forward, q, k, positions)
        params = self._parameters
        try:
            qw, kw, freq = params["q_weight"], params["k_weight"], self._buffers["_freq_bits"]
        except KeyError:                                     # a parametrised weight is no parameter of the module's own
            qw, kw, freq = self.q_weight, self.k_weight, self._freq_bits
        form = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), positions.shape,
                positions.stride(), positions.dtype, positions.get_device(), qw.shape, qw.dtype, qw.get_device(), kw.shape,
                kw.dtype, kw.get_device())
        plan = self._plans.get(form)
        if plan is None:
            plan = self._plan(form, q, k, positions, qw, kw, freq)
        if torch.is_grad_enabled():
            _hip.require_forward_only("WideHeadNormRotary", q, k, qw, kw)
        q = q if q.stride(4) == 1 else q.contiguous()
        k = k if k.stride(4) == 1 else k.contiguous()
        if not (qw.is_contiguous() and kw.is_contiguous()):
            qw, kw = qw.contiguous(), kw.contiguous()
        q_out, k_out = q.new_empty(q.shape), k.new_empty(k.shape)
        _serve.head_norm_rotary(plan, q, k, q_out, k_out, qw, kw, freq, positions, self.eps)
        return q_out, k_out

    def _plan(self, form, q: Tensor, k: Tensor, positions: Tensor, qw: Tensor, kw: Tensor, freq: Tensor):
        what = "WideHeadNormRotary"
        _hip.require_device(what, q, k, positions, qw, kw)
        for name, t in (("q", q), ("k", k)):
            if t.dim() != 5 or t.shape[0] != self.n or t.shape[4] != self.head_dim:
                raise RuntimeError(f"{what}: {name} must be [N={self.n}, B, T, heads, {self.head_dim}], got {list(t.shape)}")
        for name, t in (("q_weight", qw), ("k_weight", kw)):
            if tuple(t.shape) != (self.n, self.head_dim):
                raise RuntimeError(f"{what}: {name} must be [{self.n}, {self.head_dim}], got {list(t.shape)}")
        if q.shape[:3] != k.shape[:3]:
            raise RuntimeError(f"{what}: q {list(q.shape)} and k {list(k.shape)} differ in [N, B, T]")
        if q.dtype != k.dtype or qw.dtype != kw.dtype:
            raise RuntimeError(f"{what}: q and k, and their weights, must be of one dtype ({q.dtype}, {k.dtype}; "
                               f"{qw.dtype}, {kw.dtype})")
        if positions.dtype not in (torch.int64, torch.int32):
            raise RuntimeError(f"{what}: positions must be int32 or int64, got {positions.dtype}")
        _serve.same_device(what, q, k, positions, qw, kw, freq)
        try:
            positions = positions.expand(q.shape[:3])
        except RuntimeError:
            raise RuntimeError(f"{what}: positions {list(positions.shape)} do not broadcast to [N, B, T] "
                               f"{list(q.shape[:3])}") from None
        q = q if q.stride(4) == 1 else q.contiguous()
        k = k if k.stride(4) == 1 else k.contiguous()
        return self._plans.keep(form, _serve.head_norm_plan(q=q, k=k, q_weight=qw, positions=positions,
                                                            rotary_dim=self.rotary_dim, interleaved=self.interleaved))

    @classmethod
    def from_modules(cls, q_norms: List[nn.RMSNorm], k_norms: List[nn.RMSNorm], rotary_dim: Optional[int] = None,
                     base: float = 10000.0, interleaved: bool = False) -> "WideHeadNormRotary":
        """From the N models' nn.RMSNorm(head_dim) of queries and of keys."""
        t = q_norms[0]
        if len(q_norms) != len(k_norms) or any(tuple(m.normalized_shape) != tuple(t.normalized_shape) or m.eps != t.eps
                                               for m in (*q_norms, *k_norms)):
            raise ValueError("WideHeadNormRotary.from_modules needs as many q norms as k norms, of one shape and eps")
        if len(t.normalized_shape) != 1:
            raise ValueError("WideHeadNormRotary supports a single normalized dimension")
        weights = [m.weight for m in (*q_norms, *k_norms) if m.weight is not None]
        w = weights[0] if weights else None
        if any(x.dtype != w.dtype or x.device != w.device for x in weights):
            raise ValueError("WideHeadNormRotary.from_modules needs norms of one dtype on one device")
        # nn.RMSNorm's eps None is fp32's epsilon in 16 bits too: what it computes in
        eps = t.eps if t.eps is not None else torch.finfo(torch.float32).eps
        wide = cls(len(q_norms), t.normalized_shape[0], rotary_dim=rotary_dim, base=base, eps=eps,
                   interleaved=interleaved)
        if w is not None:
            wide = wide.to(device=w.device, dtype=w.dtype)
        with torch.no_grad():
            for dst, mods in ((wide.q_weight, q_norms), (wide.k_weight, k_norms)):
                for i, m in enumerate(mods):
                    if m.weight is not None:
                        dst[i].copy_(m.weight)
        return wide

    def __repr__(self) -> str:
        return (f"WideHeadNormRotary({self.n}x{self.head_dim}, rotary={self.rotary_dim}, base={self.base}"
                f"{', interleaved' if self.interleaved else ''})")


__all__ = ["WideHeadNormRotary"]
