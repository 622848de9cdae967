"""Plain forms in 64 bits of the operators that draw many answers to the same prompts."""

import numpy as np
import torch

from tests._serve import attend, dense


def codes_of(x):
    """8-bit codes (64 bits) and scales of rows, NaN scales where a row is not finite."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    s = torch.where(torch.isfinite(top), (top / 127).clamp_min(2.0 ** -126).float().double(), torch.full_like(top, float("nan")))
    return torch.where(torch.isnan(s), torch.zeros_like(x), torch.round(x / s)), s


def linear8(x, codes, scales, bias=None):
    """The products [n, ..., o] without the bias, and with it."""
    n, k = x.shape[0], x.shape[-1]
    c, s = codes_of(x.reshape(n, -1, k))
    y = torch.matmul(c, codes.double().transpose(1, 2).contiguous()) * s * scales.double()[:, None]
    y = y.view(*x.shape[:-1], -1)
    return y, y if bias is None else y + bias.double().view(n, *([1] * (x.dim() - 2)), -1)


def draw(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The token of one row of logits (any dtype) by the definition, the numbers as fp32 holds them."""
    x = logits.double().cpu().numpy()
    x = np.where(np.isnan(x), -np.inf, x)
    f = lambda v: np.float64(np.float32(v))  # noqa: E731
    if not (x > -np.inf).any():
        return -1
    order = np.argsort(-x, kind="stable")
    if not f(temperature) > 0:
        return int(order[0])
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp(np.where(np.isinf(x), -np.inf, x - top) / f(temperature))))
    if np.isinf(f(temperature)):
        w = np.where((x == -np.inf) | (np.isinf(top) & (x != top)), 0.0, 1.0)
    sums = np.cumsum(w[order])
    keep = len(x)
    if 0 < top_k < keep:
        keep = int(top_k)
    if top_p < 1:
        total = sums[keep - 1]
        keep = min(keep, 1 + int(np.searchsorted(sums[:keep - 1], f(top_p) * total)) if keep > 1 else 1)
    keep = min(keep, max(1, int((w[order] >= min(f(min_p), 1.0)).sum())))
    places = np.sort(order[:keep])
    sums = np.cumsum(w[places])
    u = 0.0 if not f(u) >= 2.0 ** -40 else min(f(u), 1 - 2.0 ** -24)          # numbers under 2^-40 are taken as 0
    return int(places[min(np.searchsorted(sums, u * sums[-1], side="right"), keep - 1)])


def shared(q, kp, vp, prefix_table, prefix_lens, table, lens, scale=None):
    """Pools [P, h, page, d] of values; tables and lengths on their device -> o in 64 bits, and attend()'s bound."""
    n, b = lens.shape
    share = b // prefix_lens.shape[1]
    most, own = max(int(prefix_lens.max()), 0), max(int(lens.max()), 0)
    wide = lambda t: t.repeat_interleave(share, 1)  # noqa: E731
    parts = []
    for pool in (kp, vp):
        a = wide(dense(pool.double(), prefix_table, prefix_lens, most)) if most else pool.new_zeros(n, b, 0, pool.shape[1], pool.shape[3]).double()
        c = dense(pool.double(), table, lens, own) if own else a[:, :, :0]
        # own tokens right behind the prefix's
        both = torch.zeros(n, b, most + own, *a.shape[3:], dtype=torch.float64, device=a.device)
        for i in range(n):
            for j in range(b):
                p, l = int(prefix_lens[i, j // share]), max(int(lens[i, j]), 0)
                both[i, j, :p] = a[i, j, :p]
                both[i, j, p:p + l] = c[i, j, :l]
        parts.append(both)
    total = torch.where(lens < 0, torch.zeros_like(lens), wide(prefix_lens).clamp_min(0) + lens.clamp_min(0))
    return attend(q, parts[0], parts[1], total, scale=scale)
