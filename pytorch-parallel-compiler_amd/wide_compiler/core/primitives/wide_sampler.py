"""
WideSampler: the next tokens of N models, drawn from their logits by given random numbers.

    sampler(logits [N, *batch, V], u [N, *batch])  ->  tokens int64 [N, *batch]
    w_i = exp((x_i - max x) / temperature)
    kept: the first of the order (value down, index up) such that
        there are at most top_k,
        each but the first follows less than top_p of the weight of those that top_k leaves,
        w_i >= min_p
    token = the lowest kept i with  sum of the kept w up to i  >  u * sum of all kept w

``u`` float32 in [0, 1): uniform numbers give tokens of these chances, the same numbers the same tokens.  Each model has a
temperature, a top_k, a top_p and a min_p (a number for all or one of each model); a call may give its own, as tensors
that broadcast to ``u`` (float32, int32 for top_k).  temperature <= 0 takes the most likely token, of several the one
of lowest index; top_k <= 0, top_p >= 1 and min_p <= 0 filter nothing, and the most likely token is always kept.  NaN
logits count as -infinity, which is never drawn; +infinity leaves nothing else.  A row without a logit above -infinity gives
-1.  Weights are summed exactly, as whole numbers of 2^-48 of the largest (2^-46 at 131072 logits, a bit less for every
doubling), of which each that 64 bits hold has one at least (of more than 8192 logits: each stretch of them, whose own sum is
in units of its own largest weight), so what is drawn hangs on its row alone.  ``u`` outside [0, 1)
counts as the nearest in it, under 2^-40 as 0.

The rules are read on the GPU: a captured graph replays with what they hold then.  The reference has no counterpart.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Union

import torch
from torch import Tensor, nn

from ... import _answer, _hip, _serve
from .._layout import rows_or_contiguous

_RULES = ("temperature", "top_k", "top_p", "min_p")


class WideSampler(nn.Module):
    def __init__(self, n: int, temperature: Union[float, Sequence[float]] = 1.0, top_k: Union[int, Sequence[int]] = 0,
                 top_p: Union[float, Sequence[float]] = 1.0, min_p: Union[float, Sequence[float]] = 0.0):
        super().__init__()
        self.n = n
        # [N, 4]: temperature, top_k, top_p, min_p, the floating ones as the bits of fp32, which .to(dtype) leaves as they are
        self.register_buffer("rules", torch.zeros((n, 4), dtype=torch.int32))
        self.set(temperature, top_k, top_p, min_p)
        self._plans = _serve.Plans()

    def set(self, temperature=None, top_k=None, top_p=None, min_p=None) -> None:
        """New rules, in place: a number for all models or one of each; None leaves a rule as it is.  Where one is refused, all stay
        as they were."""
        new = []
        for i, (name, rule) in enumerate(zip(_RULES, (temperature, top_k, top_p, min_p))):
            if rule is None:
                continue
            whole = name == "top_k"
            values = rule.tolist() if isinstance(rule, Tensor) else rule
            values = list(values) if isinstance(values, (list, tuple)) else [values] * self.n
            if len(values) != self.n:
                raise ValueError(f"WideSampler: {name} must be a number or {self.n} of them, got {len(values)}")
            if whole and any(not 0 <= v < 2 ** 31 or int(v) != v for v in values):
                raise ValueError(f"WideSampler: top_k must be whole numbers from 0 on, got {rule}")
            if not whole and any(math.isnan(v) or v < 0 for v in values):
                raise ValueError(f"WideSampler: {name} must not be negative, got {rule}")
            t = torch.tensor(values, dtype=torch.int32 if whole else torch.float32)
            new.append((i, t if whole else t.view(torch.int32)))
        for i, t in new:
            self.rules[:, i].copy_(t)

    def forward(self, logits: Tensor, u: Tensor, temperature: Optional[Tensor] = None, top_k: Optional[Tensor] = None,
                top_p: Optional[Tensor] = None, min_p: Optional[Tensor] = None) -> Tensor:
        if torch.compiler.is_compiling():
            return _serve.uncompiled(self.forward, logits, u, temperature, top_k, top_p, min_p)
        rules, given = self.rules, (temperature, top_k, top_p, min_p)
        form = (logits.shape, logits.stride(), logits.dtype, logits.get_device(), u.shape, u.dtype, u.get_device(),
                rules.shape, rules.dtype, rules.get_device(),
                *(None if t is None else (t.shape, t.stride(), t.dtype, t.get_device()) for t in given))
        plan = self._plans.get(form)
        if plan is None:
            plan = self._plan(form, logits, u, rules, given)
        if torch.is_grad_enabled():
            _hip.require_forward_only("WideSampler", logits)
        dense, rows, sizes, need, strides, copies = plan
        if not dense:
            logits = logits.contiguous()
        if not u.is_contiguous():
            u = u.contiguous()
        if not rules.is_contiguous():
            rules = rules.contiguous()
        if copies:
            given = tuple(t.expand(u.shape).contiguous() if t is not None and i in copies else t
                          for i, t in enumerate(given))
        tokens = torch.empty(u.shape, dtype=torch.int64, device=u.device)
        if tokens.numel():
            at = rules.data_ptr()
            _answer.sample(sizes, rows, need, logits, u, [at + 4 * i if t is None else t.data_ptr() for i, t in enumerate(given)],
                           strides, tokens)
        return tokens

    def _plan(self, form, logits: Tensor, u: Tensor, rules: Tensor, given):
        what = "WideSampler"
        if logits.dim() < 2 or logits.shape[0] != self.n or logits.shape[-1] < 1:
            raise RuntimeError(f"{what}: logits must be [N={self.n}, ..., V] of at least one logit, got {list(logits.shape)}")
        _hip.require_device(what, logits, u, rules, *given)
        if u.shape != logits.shape[:-1] or u.dtype != torch.float32:
            raise RuntimeError(f"{what}: u must be float32 {list(logits.shape[:-1])}, got {u.dtype} {list(u.shape)}")
        if tuple(rules.shape) != (self.n, 4) or rules.dtype != torch.int32:
            raise RuntimeError(f"{what}: rules must be int32 [{self.n}, 4], got {rules.dtype} {list(rules.shape)}")
        strides, copies = [], []
        for i, (name, t) in enumerate(zip(_RULES, given)):
            if t is None:
                strides += [4, 0]
                continue
            dtype = torch.int32 if name == "top_k" else torch.float32
            if t.dtype != dtype:
                raise RuntimeError(f"{what}: {name} must be {dtype}, got {t.dtype}")
            try:
                wide = t.expand(u.shape)
            except RuntimeError:
                raise RuntimeError(f"{what}: {name} {list(t.shape)} does not broadcast to {list(u.shape)}") from None
            # [N, rows] by two strides, or a copy where the batch has more of them
            dims = [(s, st) for s, st in zip(wide.shape[1:], wide.stride()[1:]) if s != 1]
            if all(a[1] == b[0] * b[1] for a, b in zip(dims, dims[1:])):
                strides += [wide.stride(0), dims[-1][1] if dims else 0]
            else:
                copies.append(i)
                strides += [math.prod(u.shape[1:]), 1]
        _serve.same_device(what, logits, u, rules, *given)
        dense, rows = rows_or_contiguous(logits)
        sizes = (_hip.dtype_code(logits.dtype, what), self.n, rows.rows, logits.shape[-1])
        return self._plans.keep(form, (dense is logits, rows, sizes, _answer.sample_workspace(sizes), tuple(strides), tuple(copies)))

    def __repr__(self) -> str:
        return f"WideSampler({self.n})"


__all__ = ["WideSampler"]
