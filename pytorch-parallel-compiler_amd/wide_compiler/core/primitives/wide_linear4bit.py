"""
WideLinear4bit: N independent linear layers with weights of 4 bits, for few rows.

    x [N, *batch, I]  ->  y [N, *batch, O],   y[i] = x[i] @ W[i].T + bias[i]
    W[i, o, k] = scale[i, o, k // group] * (code[i, o, k] - zero[i, o, k // group])

with codes of 0 to 15, groups of 32, 64 or 128 columns and zero points of 0 to 15 (8 where none are
given).  The forward (wc_linear4) brings each weight from memory once for up to 16, 32 or 64 rows (the
more weights there are, the more), so that a token's products cost what reading half a byte a weight
costs.  Whole numbers code - zero meet x, exactly, sums are fp32, and the scale multiplies each group's sum: products with
x of 2^117 and more can overflow where scaled ones would not.  An infinity in a row of x gives that row NaN in fp32, also
where the formula has an infinity.

The buffers hold the weights as the kernel reads them (``packed`` [N, O / 16, I / 128, 64, 4] int32,
``scales`` and ``zeros`` [N, O / 16, groups, 16], sizes rounded up); ``from_codes`` packs them from
rows and ``from_modules`` quantises WideLinear's modules; ``dequantize()`` gives the weights they
stand for.  The reference has no counterpart.
"""

from __future__ import annotations

from typing import List, Optional

import torch
from torch import Tensor, nn

from ... import _hip, _serve
from .._layout import rows_or_contiguous

# column e of a lane's 8 stands in this nibble of its word
_NIBBLE = (0, 4, 1, 5, 2, 6, 3, 7)


class WideLinear4bit(nn.Module):
    def __init__(self, n: int, in_features: int, out_features: int, group_size: int = 128, bias: bool = True,
                 dtype: torch.dtype = torch.float32):
        super().__init__()
        if group_size not in (32, 64, 128):
            raise ValueError(f"WideLinear4bit: group_size must be 32, 64 or 128, got {group_size}")
        if in_features < 1:
            raise ValueError("WideLinear4bit: in_features must be positive")
        _hip.dtype_code(dtype, "WideLinear4bit")
        self.n = n
        self.in_features = in_features
        self.out_features = out_features
        self.group_size = group_size
        rt, kt = -(-out_features // 16), -(-in_features // 128)
        meta = (n, rt, kt * (128 // group_size), 16)
        self.register_buffer("packed", torch.zeros((n, rt, kt, 64, 4), dtype=torch.int32))
        self.register_buffer("scales", torch.zeros(meta, dtype=dtype))
        self.register_buffer("zeros", torch.full(meta, 8, dtype=torch.uint8))
        self.register_buffer("bias", torch.zeros((n, out_features), dtype=dtype) if bias else None)
        self._plans = _serve.Plans()

    def forward(self, x: Tensor) -> Tensor:
        if torch.compiler.is_compiling():
            return _serve.uncompiled(self.forward, x)
        bufs = self._buffers
        try:
            packed, scales, zeros, bias = bufs["packed"], bufs["scales"], bufs["zeros"], bufs["bias"]
        except KeyError:                                     # one that was parametrised, or became something else
            packed, scales, zeros, bias = self.packed, self.scales, self.zeros, self.bias
        form = (x.shape, x.stride(), x.dtype, x.get_device(), packed.shape, packed.dtype, packed.get_device(), scales.shape,
                scales.dtype, scales.get_device(), zeros.shape, zeros.dtype, zeros.get_device(),
                None if bias is None else (bias.shape, bias.dtype, bias.get_device()))
        plan = self._plans.get(form)
        if plan is None:
            plan = self._plan(form, x, packed, scales, zeros, bias)
        if torch.is_grad_enabled():
            _hip.require_forward_only("WideLinear4bit", x, scales, bias)
        dense, rows, sizes, shape = plan
        if not dense:
            x = x.contiguous()
        if not (packed.is_contiguous() and scales.is_contiguous() and zeros.is_contiguous()):
            packed, scales, zeros = packed.contiguous(), scales.contiguous(), zeros.contiguous()
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        y = x.new_empty(shape)
        if y.numel():
            _serve.linear4(sizes, rows, x, packed, scales, zeros, bias, y)
        return y

    def _plan(self, form, x: Tensor, packed: Tensor, scales: Tensor, zeros: Tensor, bias: Optional[Tensor]):
        what = "WideLinear4bit"
        if x.dim() < 2 or x.shape[0] != self.n or x.shape[-1] != self.in_features:
            raise RuntimeError(f"{what}: expected input [N={self.n}, ..., {self.in_features}], got {list(x.shape)}")
        _hip.require_device(what, x, packed)
        if x.dtype != scales.dtype or (bias is not None and bias.dtype != x.dtype):
            raise RuntimeError(f"{what}: input dtype {x.dtype} != {scales.dtype} of scales and bias")
        rt, kt = -(-self.out_features // 16), -(-self.in_features // 128)
        meta = (self.n, rt, kt * (128 // self.group_size), 16)
        for name, t, shape, dtype in (("packed", packed, (self.n, rt, kt, 64, 4), torch.int32), ("scales", scales, meta, x.dtype),
                                      ("zeros", zeros, meta, torch.uint8), ("bias", bias, (self.n, self.out_features), x.dtype)):
            if t is not None and (t.dtype != dtype or tuple(t.shape) != shape):
                raise RuntimeError(f"{what}: {name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
        _serve.same_device(what, x, packed, scales, zeros, bias)
        dense, rows = rows_or_contiguous(x)
        sizes = (_hip.dtype_code(x.dtype, "linear4"), self.group_size, self.n, rows.rows, self.out_features, self.in_features)
        return self._plans.keep(form, (dense is x, rows, sizes, (*x.shape[:-1], self.out_features)))

    def _pack(self, i: int, codes: Tensor, scales: Tensor, zeros: Optional[Tensor]) -> None:
        """codes [O, I] uint8 of 0-15, scales and zeros [O, ceil(I / group)] into model i's part of the buffers: one model
        at a time, because that takes some bytes a weight on the way."""
        rt, kt = self.packed.shape[1:3]
        full = torch.zeros((rt * 16, kt * 128), dtype=torch.uint8, device=codes.device)
        full[:self.out_features, :self.in_features] = codes
        # [row tile, row, column tile, word, lane group, column] -> [.., lane group, row, word, column]
        c = full.view(rt, 16, kt, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)
        half = torch.empty((*c.shape[:-1], 8), dtype=torch.uint8, device=codes.device)
        half[..., list(_NIBBLE)] = c
        words = half[..., 0::2] | (half[..., 1::2] << 4)                 # bytes, the low nibble first
        self.packed[i].copy_(words.contiguous().view(torch.int32).view(self.packed.shape[1:]))
        for dst, src in ((self.scales[i], scales), (self.zeros[i], zeros)):
            if src is not None:
                rows = torch.zeros((rt * 16, dst.shape[1]), dtype=dst.dtype, device=codes.device)
                rows[:self.out_features, :src.shape[1]] = src
                dst.copy_(rows.view(rt, 16, -1).transpose(1, 2))

    @classmethod
    def from_codes(cls, codes: Tensor, scales: Tensor, *, in_features: int, group_size: int = 128,
                   zeros: Optional[Tensor] = None, bias: Optional[Tensor] = None) -> "WideLinear4bit":
        """codes [N, O, ceil(I / 2)] uint8, two to a byte, the even column in the low half; scales
        [N, O, ceil(I / group)] of the dtype of the inputs; zeros the same of uint8 (0 to 15) or None; bias [N, O]."""
        what = "WideLinear4bit.from_codes"
        if group_size not in (32, 64, 128):
            raise ValueError(f"{what}: group_size must be 32, 64 or 128, got {group_size}")
        if codes.dim() != 3 or codes.dtype != torch.uint8 or codes.shape[2] != (in_features + 1) // 2:
            raise ValueError(f"{what}: codes must be uint8 [N, O, {(in_features + 1) // 2}], got {codes.dtype} {list(codes.shape)}")
        meta = (*codes.shape[:2], -(-in_features // group_size))
        if tuple(scales.shape) != meta or (zeros is not None and (tuple(zeros.shape) != meta or zeros.dtype != torch.uint8)):
            raise ValueError(f"{what}: scales and uint8 zeros must be {list(meta)}")
        if bias is not None and tuple(bias.shape) != tuple(codes.shape[:2]):
            raise ValueError(f"{what}: bias must be {list(codes.shape[:2])}, got {list(bias.shape)}")
        if zeros is not None and zeros.numel() and int(zeros.max()) > 15:
            raise ValueError(f"{what}: zero points must be within [0, 15]")
        wide = cls(codes.shape[0], in_features, codes.shape[1], group_size, bias=bias is not None,
                   dtype=scales.dtype).to(codes.device)
        with torch.no_grad():
            for i, c in enumerate(codes):
                rows = torch.stack((c & 15, c >> 4), -1).flatten(-2)[:, :in_features]
                wide._pack(i, rows, scales[i], None if zeros is None else zeros[i])
            if bias is not None:
                wide.bias.copy_(bias)
        return wide

    @classmethod
    def from_modules(cls, modules: List[nn.Linear], group_size: int = 128) -> "WideLinear4bit":
        """Quantises N nn.Linear: each group's codes span its values and zero, code = round(w / scale) + zero."""
        t = modules[0]
        form = lambda m: (tuple(m.weight.shape), m.weight.dtype, m.weight.device,  # noqa: E731
                          None if m.bias is None else (m.bias.dtype, m.bias.device))
        if any(form(m) != form(t) for m in modules):
            raise ValueError("WideLinear4bit.from_modules needs modules of one shape, dtype and device, all with a bias or all "
                             "without")
        o, k = t.out_features, t.in_features
        wide = cls(len(modules), k, o, group_size, bias=t.bias is not None, dtype=t.weight.dtype).to(t.weight.device)
        groups, info = -(-k // group_size), torch.finfo(t.weight.dtype)
        with torch.no_grad():
            for i, m in enumerate(modules):
                w = torch.nn.functional.pad(m.weight.float(), (0, groups * group_size - k)).view(o, groups, group_size)
                lo, hi = w.amin(-1).clamp_max(0), w.amax(-1).clamp_min(0)
                # a step, under the type's normal values rounded up (to the nearest it may be half as large, or 0); 1 of zeros
                step, least = hi.double() / 15 - lo.double() / 15, info.tiny * info.eps
                step = torch.where(step < info.tiny, torch.ceil(step / least) * least, step)
                scales = torch.where(step == 0, 1.0, step).to(t.weight.dtype)
                s = scales.float()
                zeros = torch.round(-lo / s).clamp(0, 15)
                codes = (torch.round(w / s[..., None]) + zeros[..., None]).clamp(0, 15)
                wide._pack(i, codes.to(torch.uint8).flatten(-2)[:, :k], scales, zeros.to(torch.uint8))
                if m.bias is not None:
                    wide.bias[i].copy_(m.bias)
        return wide

    def dequantize(self) -> Tensor:
        """The weights the codes stand for, float32 [N, O, I]."""
        n, rt, kt = self.packed.shape[:3]
        b = self.packed.contiguous().view(torch.uint8).view(n, rt, kt, 4, 16, 4, 4)
        half = torch.stack((b & 15, b >> 4), -1).flatten(-2)             # nibbles in order
        c = half[..., list(_NIBBLE)].permute(0, 1, 4, 2, 5, 3, 6).reshape(n, rt * 16, kt * 128)
        rows = lambda t: t.transpose(2, 3).reshape(n, rt * 16, -1).float().repeat_interleave(self.group_size, -1)  # noqa: E731
        w = (c.float() - rows(self.zeros)) * rows(self.scales)
        return w[:, :self.out_features, :self.in_features]

    def __repr__(self) -> str:
        return (f"WideLinear4bit({self.n}x[{self.in_features}->{self.out_features}], group={self.group_size})")


__all__ = ["WideLinear4bit"]
