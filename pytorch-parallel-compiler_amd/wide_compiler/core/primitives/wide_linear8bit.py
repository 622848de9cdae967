"""
WideLinear8bit: N independent linear layers in 8-bit integers, for prompts and batches as for single tokens.

    x [N, *batch, I]  ->  y [N, *batch, O]
    s = max(max |x| / 127, 2^-126) of each row,  c = x / s to the nearest, ties to even
    y[i, r, o] = s[i, r] scale[i, o] sum_k c[i, r, k] code[i, o, k] + bias[i, o]

with codes of -127 to 127 and a scale for every output (channel) of every model.  The rows of x get their codes inside
the call (wc_linear8); sums are exact in 32-bit integers, so a row's result depends neither on the other rows nor on how
the work is split.  A row with an infinity or NaN gives NaN.  Inputs of at most 131072 columns.

The buffers hold the weights as the kernel reads them (``packed`` [N, O / 16, I / 64, 64, 16] int8, columns rounded up to
128; ``scale_bits`` [N, O], the scales as the bits of fp32, which ``.to(dtype)`` leaves as they are); ``from_codes`` packs
them from rows, ``from_modules`` quantises WideLinear's modules and ``dequantize()`` gives the weights they stand for.
The reference has no counterpart.
"""

from __future__ import annotations

from typing import List, Optional

import torch
from torch import Tensor, nn

from ... import _answer, _hip, _serve
from .._layout import rows_or_contiguous

_MOST = float.fromhex("0x1.020406p121")          # the largest scale: 127 of the next one round to infinity in fp32


class WideLinear8bit(nn.Module):
    def __init__(self, n: int, in_features: int, out_features: int, bias: bool = True, dtype: torch.dtype = torch.float32):
        """dtype: of the bias; inputs have its dtype, and any of the supported ones where there is none."""
        super().__init__()
        if not 1 <= in_features <= 131072:
            raise ValueError(f"WideLinear8bit: in_features must be within [1, 131072], got {in_features}")
        _hip.dtype_code(dtype, "WideLinear8bit")
        self.n = n
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("packed", torch.zeros(self._packed_shape(), dtype=torch.int8))
        self.register_buffer("scale_bits", torch.zeros((n, out_features), dtype=torch.int32))
        self.register_buffer("bias", torch.zeros((n, out_features), dtype=dtype) if bias else None)
        self._plans = _serve.Plans()

    def _packed_shape(self):
        return self.n, -(-self.out_features // 16), -(-self.in_features // 128) * 2, 64, 16

    @property
    def scales(self) -> Tensor:
        return self.scale_bits.view(torch.float32)

    def forward(self, x: Tensor) -> Tensor:
        if torch.compiler.is_compiling():
            return _serve.uncompiled(self.forward, x)
        bufs = self._buffers
        try:
            packed, scales, bias = bufs["packed"], bufs["scale_bits"], bufs["bias"]
        except KeyError:                                     # one that was parametrised, or became something else
            packed, scales, bias = self.packed, self.scale_bits, self.bias
        form = (x.shape, x.stride(), x.dtype, x.get_device(), packed.shape, packed.dtype, packed.get_device(), scales.shape,
                scales.dtype, scales.get_device(), None if bias is None else (bias.shape, bias.dtype, bias.get_device()))
        plan = self._plans.get(form)
        if plan is None:
            plan = self._plan(form, x, packed, scales, bias)
        if torch.is_grad_enabled():
            _hip.require_forward_only("WideLinear8bit", x, bias)
        dense, rows, sizes, need, shape = plan
        if not dense:
            x = x.contiguous()
        if not (packed.is_contiguous() and scales.is_contiguous()):
            packed, scales = packed.contiguous(), scales.contiguous()
        if bias is not None and not bias.is_contiguous():
            bias = bias.contiguous()
        y = x.new_empty(shape)
        if y.numel():
            _answer.linear8(sizes, rows, need, x, packed, scales, bias, y)
        return y

    def _plan(self, form, x: Tensor, packed: Tensor, scales: Tensor, bias: Optional[Tensor]):
        what = "WideLinear8bit"
        if x.dim() < 2 or x.shape[0] != self.n or x.shape[-1] != self.in_features:
            raise RuntimeError(f"{what}: expected input [N={self.n}, ..., {self.in_features}], got {list(x.shape)}")
        _hip.require_device(what, x, packed)
        if bias is not None and bias.dtype != x.dtype:
            raise RuntimeError(f"{what}: input dtype {x.dtype} != {bias.dtype} of the bias")
        for name, t, shape, dtype in (("packed", packed, self._packed_shape(), torch.int8),
                                      ("scale_bits", scales, (self.n, self.out_features), torch.int32),
                                      ("bias", bias, (self.n, self.out_features), x.dtype)):
            if t is not None and (t.dtype != dtype or tuple(t.shape) != shape):
                raise RuntimeError(f"{what}: {name} must be {dtype} {list(shape)}, got {t.dtype} {list(t.shape)}")
        _serve.same_device(what, x, packed, scales, bias)
        dense, rows = rows_or_contiguous(x)
        sizes = (_hip.dtype_code(x.dtype, what), self.n, rows.rows, self.out_features, self.in_features)
        return self._plans.keep(form, (dense is x, rows, sizes, _answer.linear8_workspace(sizes),
                                       (*x.shape[:-1], self.out_features)))

    def _pack(self, i: int, codes: Tensor) -> None:
        """codes [O, I] int8 into model i's part of ``packed``."""
        rt, kt = self.packed.shape[1:3]
        full = torch.zeros((rt * 16, kt * 64), dtype=torch.int8, device=codes.device)
        full[:self.out_features, :self.in_features] = codes
        # [row tile, row, column tile, lane group, column] -> [row tile, column tile, lane group, row, column]
        self.packed[i].copy_(full.view(rt, 16, kt, 4, 16).permute(0, 2, 3, 1, 4).reshape(rt, kt, 64, 16))

    def _set_scales(self, i: int, scales: Tensor) -> None:
        self.scale_bits[i].copy_(scales.float().contiguous().view(torch.int32))

    @classmethod
    def from_codes(cls, codes: Tensor, scales: Tensor, bias: Optional[Tensor] = None) -> "WideLinear8bit":
        """codes [N, O, I] int8 of -127 to 127; scales float32 [N, O]; bias [N, O] of the inputs' dtype."""
        what = "WideLinear8bit.from_codes"
        if codes.dim() != 3 or codes.dtype != torch.int8:
            raise ValueError(f"{what}: codes must be int8 [N, O, I], got {codes.dtype} {list(codes.shape)}")
        if tuple(scales.shape) != tuple(codes.shape[:2]) or scales.dtype != torch.float32:
            raise ValueError(f"{what}: scales must be float32 {list(codes.shape[:2])}, got {scales.dtype} {list(scales.shape)}")
        if bias is not None and tuple(bias.shape) != tuple(codes.shape[:2]):
            raise ValueError(f"{what}: bias must be {list(codes.shape[:2])}, got {list(bias.shape)}")
        if codes.numel() and int(codes.min()) < -127:
            raise ValueError(f"{what}: codes must be within [-127, 127]")
        n, o, k = codes.shape
        wide = cls(n, k, o, bias=bias is not None, dtype=torch.float32 if bias is None else bias.dtype).to(codes.device)
        with torch.no_grad():
            for i in range(n):
                wide._pack(i, codes[i])
                wide._set_scales(i, scales[i])
            if bias is not None:
                wide.bias.copy_(bias)
        return wide

    @classmethod
    def from_modules(cls, modules: List[nn.Linear]) -> "WideLinear8bit":
        """Quantises N nn.Linear: scale = max |w| / 127 of each output's weights (a step less for fp32's largest value), code =
        w / scale to the nearest."""
        t = modules[0]
        form = lambda m: (tuple(m.weight.shape), m.weight.dtype, m.weight.device,  # noqa: E731
                          None if m.bias is None else (m.bias.dtype, m.bias.device))
        if any(form(m) != form(t) for m in modules):
            raise ValueError("WideLinear8bit.from_modules needs modules of one shape, dtype and device, all with a bias or all "
                             "without")
        wide = cls(len(modules), t.in_features, t.out_features, bias=t.bias is not None, dtype=t.weight.dtype).to(t.weight.device)
        with torch.no_grad():
            for i, m in enumerate(modules):
                w = m.weight.double()
                top = w.abs().amax(-1)
                s = (top / 127).clamp_min(2.0 ** -126).float()
                s = torch.where(torch.isfinite(top), s.clamp_max(_MOST), s)
                wide._pack(i, torch.round(w / s.double()[:, None]).clamp(-127, 127).to(torch.int8))
                wide._set_scales(i, s)
                if m.bias is not None:
                    wide.bias[i].copy_(m.bias)
        return wide

    def dequantize(self) -> Tensor:
        """The weights the codes stand for, float32 [N, O, I]."""
        n, rt, kt = self.packed.shape[:3]
        c = self.packed.view(n, rt, kt, 4, 16, 16).permute(0, 1, 4, 2, 3, 5).reshape(n, rt * 16, kt * 64)
        return c[:, :self.out_features, :self.in_features].float() * self.scales[..., None]

    def __repr__(self) -> str:
        return f"WideLinear8bit({self.n}x[{self.in_features}->{self.out_features}])"


__all__ = ["WideLinear8bit"]
