"""Plain forms in 64 bits of the decode-step operators, and inputs for them."""

import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}    # half a rounding step


def within(got, ref, rel, absolute):
    """|got - ref| <= rel |ref| + absolute everywhere (absolute a number or a tensor that broadcasts), and half a step
    of got's subnormal values: under the smallest normal value the step no longer shrinks with the value (fp16: values
    under 2^-14 are 2^-24 apart, so a correct rounding is off by up to 2^-25)."""
    if got.dtype in HALF:
        absolute = absolute + torch.finfo(got.dtype).tiny * HALF[got.dtype]
    got, ref = got.double(), ref.double()
    inf = torch.isinf(ref)
    bad = torch.where(inf, got != ref, (got - ref).abs() > rel * ref.abs() + absolute) | (torch.isnan(got) != torch.isnan(ref))
    assert not bad.any(), (int(bad.sum()), (got - ref).abs().max().item(), bad.nonzero()[:4].tolist())


def quantise(x):
    """Codes and scales of rows (last dim), and the values they stand for, in 64 bits."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    s = torch.where(torch.isfinite(top), (top / 127).clamp_min(2.0 ** -126).float().double(),
                    torch.full_like(top, float("nan")))
    return torch.round(x / s) * s


def make_table(lens, page, gen, extra=2, width=None):
    """Block table [n, b, m] (int32, -1 behind the last page) of random distinct pages for lengths lens [n, b]."""
    n, b = lens.shape
    need = (lens + page - 1) // page
    m = max(int(need.max()), 1) if width is None else width
    total = int(need.sum()) + extra
    ids = torch.randperm(total, generator=gen).to(torch.int32)
    table = torch.full((n, b, m), -1, dtype=torch.int32)
    at = 0
    for i in range(n):
        for k in range(b):
            c = int(need[i, k])
            table[i, k, :c] = ids[at:at + c]
            at += c
    return table, total


def dense(pages, table, lens, most):
    """Rows [n, b, most, h, row] of a pool [P, h, page, row] (zeros from a length on), on the pool's device."""
    page = pages.shape[2]
    at = torch.arange(most, device=pages.device)
    block = (at // page).clamp_max(table.shape[2] - 1)
    ids = table.long()[:, :, block].clamp(0, pages.shape[0] - 1)
    x = pages.transpose(1, 2)[ids, at % page]
    return torch.where((at < lens.long()[..., None])[..., None, None], x, torch.zeros_like(x))


def attend(q, k, v, lens, first=None, scale=None):
    """q [n, b, hq, d], k / v [n, b, L, hkv, d] in 64 bits -> o, and the largest sum |q k| of a score."""
    n, b, hq, d = q.shape
    hkv, length = k.shape[3], k.shape[2]
    q, k, v = q.double(), k.double(), v.double()
    k, v = (t.permute(0, 1, 3, 2, 4).repeat_interleave(hq // hkv, 2) for t in (k, v))        # [n, b, hq, L, d]
    scale = d ** -0.5 if scale is None else scale
    prod = q[:, :, :, None] * k
    s = prod.sum(-1) * scale
    at = torch.arange(length, device=q.device)
    has = at < lens.long()[..., None]
    if first is not None:
        has &= at >= first.long()[..., None]
    has = has[:, :, None]
    s = torch.where(has, s, -torch.inf)
    some = has.any(-1, keepdim=True)
    p = torch.softmax(torch.where(some, s, 0.0), -1)
    v = torch.where(has[..., None], v, 0.0)
    o = torch.where(some[..., None], (p[..., None] * v), 0.0).sum(-2)
    big = torch.where(has, prod.abs().sum(-1), 0.0).nan_to_num(0, 0, 0).amax().item() * abs(scale) if length else 0.0
    return o, big


def attend_slack(dtype, big, d, length, vmax, planes=2.0 ** -16):
    """What fp32 arithmetic may add to the rounding of the result: a score is off by (d + 4) 2^-24 of its sum of
    magnitudes, its exponential by that twice over (numerator and sum) and 2^-21, the sums by length 2^-24 each, P by
    its planes' last bit; each of the largest value."""
    return vmax * (2 * (d + 4) * 2.0 ** -24 * big + 2.0 ** -20 + 2 * length * 2.0 ** -24 +
                   (planes if dtype != torch.float32 else 0.0))
