"""
Operators of a decode step, by which their speed is followed: an ensemble of N decoders answers
token by token.

  norm       RMS norm of every query and key head with the rotation by position in the same pass
  cache      writing a paged key-value cache, as it is or in 8 bits, and reading it back
  attention  one new token of every sequence over its pages
  linear4    products with weights of 4 bits and group scales, for few rows

`listed()` holds the fixed cases, `draw(rng)` samples the ranges they stand for:

  norm       1-16 models, 1-16 sequences, 1-4096 tokens each, 1-32 query heads over 1-32 key heads of
             32-256, whole or partial rotation, both pairings, positions up to a million
  cache      1-64 sequences of 1-2048 new tokens at any offset, pages of 8-128 tokens, 1-16 heads of
             32-256, in the tensors' type or in 8 bits
  attention  1-128 sequences of 1-131072 cached tokens, pages of 8-128, 1-16 query heads to a key
             head, heads of 32-256, whole or windowed, in the tensors' type or in 8 bits
  linear4    1-16 models, 1-64 rows, widths 64-8192, groups of 32, 64 or 128, with and without zero points

all of them in fp32, bf16 and fp16.
"""

import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _wc():
    pkg = os.path.join(_ROOT, "pytorch-parallel-compiler_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import wide_compiler
    return wide_compiler


def listed():
    return [
        # one token of 32 sequences: the call between the projections and the cache, where latency counts
        dict(name="norm_token_bf16", kind="norm", dtype="bf16", n=8, b=4, t=1, hq=32, hkv=8, dh=128, rot=128,
             interleaved=False, far=100000),
        # prompts of 2048 tokens before their attention: memory traffic
        dict(name="norm_prompt_bf16", kind="norm", dtype="bf16", n=4, b=2, t=2048, hq=32, hkv=8, dh=128, rot=128,
             interleaved=False, far=8192),
        # an odd number of tokens, heads of 80 of which half rotate, neighbours paired, fp32
        dict(name="norm_ragged_f32", kind="norm", dtype="f32", n=3, b=5, t=333, hq=12, hkv=2, dh=80, rot=40,
             interleaved=True, far=1000000),
        # the new token of 32 sequences goes to the cache as it is
        dict(name="cache_token_bf16", kind="cache", dtype="bf16", n=8, b=4, t=1, hkv=8, dh=128, page=16, bits=16,
             past=300),
        # prompts of unequal length go to an 8-bit cache and are read back for the next chunk
        dict(name="cache_prompt_int8", kind="cache", dtype="bf16", n=4, b=4, t=1500, hkv=8, dh=128, page=32, bits=8,
             past=100),
        # the first answer of one short conversation: latency
        dict(name="attend_short_bf16", kind="attention", dtype="bf16", n=1, b=1, len=257, hq=32, hkv=8, dh=128, page=16,
             bits=16, window=0),
        # a batch of conversations of unequal length over an 8-bit cache
        dict(name="attend_batch_int8", kind="attention", dtype="bf16", n=4, b=16, len=4000, hq=32, hkv=8, dh=128, page=16,
             bits=8, window=0),
        # two documents of 131072 tokens: split over the length
        dict(name="attend_long_bf16", kind="attention", dtype="bf16", n=1, b=2, len=131072, hq=32, hkv=8, dh=128,
             page=64, bits=16, window=0),
        # an ensemble of small fp32 models with as many key heads as query heads, an odd page size
        dict(name="attend_heads_f32", kind="attention", dtype="f32", n=8, b=4, len=777, hq=8, hkv=8, dh=64, page=24,
             bits=32, window=0),
        # one token through one square layer of each of four models: matrix-vector products
        dict(name="linear4_token_bf16", kind="linear4", dtype="bf16", n=4, m=1, k=4096, o=4096, group=128, zeros=False),
        # small fp32 models, a width that ends inside a group
        dict(name="linear4_odd_f32", kind="linear4", dtype="f32", n=6, m=5, k=1000, o=500, group=32, zeros=True),
        # the widening layer for a batch of 64 rows
        dict(name="linear4_batch_f16", kind="linear4", dtype="f16", n=8, m=64, k=2048, o=8192, group=64, zeros=True),
    ]


# ---------------------------------------------------------------------------------------
# drawn cases
# ---------------------------------------------------------------------------------------

def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer's width: mostly a multiple of 16, now and then any number."""
    w = _log(rng, lo, hi)
    return w if rng.random() < 0.25 else max(lo, (w + 8) // 16 * 16)


def _draw_one(rng):
    kind = rng.choice(["norm", "cache", "attention", "attention", "linear4", "linear4"])
    dt = rng.choice(["f32", "bf16", "bf16", "f16"])
    dh = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    bits = rng.choice([8, {"f32": 32}.get(dt, 16)])
    if kind == "norm":
        hkv = rng.choice([1, 2, 4, 8])
        return dict(kind=kind, dtype=dt, n=_log(rng, 1, 16), b=_log(rng, 1, 16), t=_log(rng, 1, 4096),
                    hq=hkv * rng.choice([1, 2, 3, 4]), hkv=hkv, dh=dh, rot=rng.choice([dh, dh, dh // 2]),
                    interleaved=rng.random() < 0.4, far=_log(rng, 16, 1000000))
    if kind == "cache":
        return dict(kind=kind, dtype=dt, n=_log(rng, 1, 8), b=_log(rng, 1, 8), t=_log(rng, 1, 2048),
                    hkv=rng.choice([1, 2, 4, 8, 16]), dh=dh, page=page, bits=bits, past=_log(rng, 1, 1000))
    if kind == "attention":
        hkv = rng.choice([1, 2, 4, 8])
        length = _log(rng, 1, 131072)
        return dict(kind=kind, dtype=dt, n=_log(rng, 1, 8), b=_log(rng, 1, 16), len=length,
                    hq=hkv * rng.choice([1, 1, 2, 3, 4, 7, 8, 16]), hkv=hkv, dh=dh, page=page, bits=bits,
                    window=rng.choice([0, 0, 0, _log(rng, 1, length)]))
    return dict(kind=kind, dtype=dt, n=_log(rng, 1, 16), m=_log(rng, 1, 64), k=_width(rng, 64, 8192),
                o=_width(rng, 64, 8192), group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        t = top.setdefault(c["kind"], [0, 0])
        t[0], t[1] = max(t[0], w["bytes"]), max(t[1], w["flops"])
    while True:
        c = _draw_one(rng)
        w = work(c)
        if w["bytes"] <= top[c["kind"]][0] and w["flops"] <= top[c["kind"]][1]:
            return c


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------

def _lengths(c):
    """The cached lengths of a case's sequences, longest first: from a quarter of the longest up; with 16
    sequences or more, one has a single token and one has none."""
    n, top = c["n"] * c["b"], c["len"]
    lens = [max(1, top - i * (3 * top // 4) // max(n - 1, 1)) for i in range(n)]
    if n >= 16:
        lens[-2:] = [1, 0]
    return lens


def _counts(c):
    """The new tokens of a case's sequences: from half of the most up."""
    n, top = c["n"] * c["b"], c["t"]
    return [max(1, top - i * (top // 2) // max(n - 1, 1)) for i in range(n)]


def _starts(c):
    """The tokens that a case's sequences have already: from none to the most."""
    n = c["n"] * c["b"]
    return [i * c["past"] // max(n - 1, 1) for i in range(n)]


def _shuffled(values, seed):
    values = list(values)
    random.Random(seed).shuffle(values)
    return values


def _table(need, most, page, gen, c):
    """A block table [N, B, M] of distinct pages of a pool in random order, -1 behind each sequence's last."""
    pages = [-(-x // page) for x in need]
    m = max(pages + [1])
    ids = torch.randperm(most, generator=gen, device=DEV).to(torch.int32).tolist()
    rows, at = [], 0
    for p in pages:
        rows.append(ids[at:at + p] + [-1] * (m - p))
        at += p
    return torch.tensor(rows, dtype=torch.int32, device=DEV).view(c["n"], c["b"], m)


def _ints(values, c):
    return torch.tensor(values, dtype=torch.int32, device=DEV).view(c["n"], c["b"])


def _quantise(x):
    """8-bit codes and fp32 scales of rows: s = max(max |x| / 127, 2^-126), code = x / s to the nearest, ties to
    even; in 64 bits, because a quotient next to a half decides a code."""
    x = x.double()
    s = (x.abs().amax(-1) / 127).clamp_min(2.0 ** -126).float()
    return torch.round(x / s.double()[..., None]).to(torch.int8), s


def _pool(pages, c, gen):
    """One pool of pages [P, Hkv, page, Dh] (and its scales [P, Hkv, page]) holding values of unit size."""
    shape = (pages, c["hkv"], c["page"], c["dh"])
    x = torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(DTYPES[c["dtype"]])
    return (x, None) if c["bits"] != 8 else _quantise(x)


def prepare(case, seed):
    c, kind, dt = case, case["kind"], DTYPES[case["dtype"]]
    gen = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32)  # noqa: E731
    st = dict(kind=kind, case=c)
    if kind == "norm":
        # q and k as the projections leave them: columns of one [N, B, T, (Hq + 2 Hkv) Dh] tensor
        hq, hkv, dh = c["hq"], c["hkv"], c["dh"]
        qkv = (rand(c["n"], c["b"], c["t"], (hq + 2 * hkv) * dh) * 3).to(dt)
        st["q"] = qkv[..., :hq * dh].unflatten(-1, (hq, dh))
        st["k"] = qkv[..., hq * dh:(hq + hkv) * dh].unflatten(-1, (hkv, dh))
        first = torch.randint(0, c["far"], (c["n"], c["b"], 1), generator=gen, device=DEV)
        st["positions"] = first + torch.arange(c["t"], device=DEV)
        st["q_weight"], st["k_weight"] = ((1 + 0.1 * rand(c["n"], dh)).to(dt) for _ in range(2))
        st["base"], st["eps"] = 10000.0, 1e-6
        if own:
            mod = _wc().WideHeadNormRotary(c["n"], dh, rotary_dim=c["rot"], base=st["base"], eps=st["eps"],
                                           interleaved=c["interleaved"]).to(device=DEV, dtype=dt)
            with torch.no_grad():
                mod.q_weight.copy_(st["q_weight"])
                mod.k_weight.copy_(st["k_weight"])
            st["module"] = mod
    elif kind == "cache":
        start, count = _shuffled(_starts(c), seed), _shuffled(_counts(c), seed + 1)
        need = [s + t for s, t in zip(start, count)]
        pages = len(need) * -(-(c["past"] + c["t"]) // c["page"]) + 3           # some of them are no one's
        st["table"] = _table(need, pages, c["page"], gen, c)
        st["start"], st["count"], st["lengths"] = _ints(start, c), _ints(count, c), _ints(need, c)
        st["max_length"] = c["past"] + c["t"]
        st["k"], st["v"] = (rand(c["n"], c["b"], c["t"], c["hkv"], c["dh"]).to(dt) for _ in range(2))
        for name in ("k", "v"):
            st[name + "_pages"], st[name + "_scales"] = _pool(pages, c, gen)
    elif kind == "attention":
        need = _shuffled(_lengths(c), seed)
        pages = sum(-(-x // c["page"]) for x in need) + 3
        st["table"] = _table(need, pages, c["page"], gen, c)
        st["lengths"] = _ints(need, c)
        st["first"] = _ints([max(x - c["window"], 0) for x in need], c) if c["window"] else None
        st["q"] = rand(c["n"], c["b"], c["hq"], c["dh"]).to(dt)
        for name in ("k", "v"):
            st[name + "_pages"], st[name + "_scales"] = _pool(pages, c, gen)
    else:
        n, m, k, o, g = c["n"], c["m"], c["k"], c["o"], -(-c["k"] // c["group"])
        # two codes a byte, the even column in the low half
        st["codes"] = torch.randint(0, 256, (n, o, (k + 1) // 2), generator=gen, device=DEV, dtype=torch.uint8)
        st["scales"] = ((0.5 + torch.rand((n, o, g), generator=gen, device=DEV)) * (0.2 / math.sqrt(k))).to(dt)
        st["zeros"] = (torch.randint(5, 11, (n, o, g), generator=gen, device=DEV, dtype=torch.uint8)
                       if c["zeros"] else None)
        st["x"] = rand(n, m, k).to(dt)
        if own:
            st["module"] = _wc().WideLinear4bit.from_codes(st["codes"], st["scales"], in_features=k,
                                                           group_size=c["group"], zeros=st["zeros"])
    if own and kind in ("cache", "attention"):
        st["cache"] = _wc().WidePagedCache.from_pages(st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"],
                                                      dtype=dt)
    return st


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------

def run(state):
    st, kind = state, state["kind"]
    if own:
        with torch.no_grad():
            if kind == "norm":
                return st["module"](st["q"], st["k"], st["positions"])
            if kind == "cache":
                cache = st["cache"]
                cache.write(st["k"], st["v"], st["table"], st["start"], st["count"])
                if st["case"]["bits"] == 8:
                    return cache.read(st["table"], st["lengths"], st["max_length"])
                return cache.k_pages, cache.v_pages
            if kind == "attention":
                return st["cache"].attend(st["q"], st["table"], st["lengths"], first=st["first"])
            return st["module"](st["x"])
    return {"norm": _plain_norm, "cache": _plain_cache, "attention": _plain_attention,
            "linear4": _plain_linear4}[kind](st)


def _plain_norm(st):
    c, rot = st["case"], st["case"]["rot"]
    freq = st["base"] ** (-torch.arange(0, rot, 2, device=DEV, dtype=torch.float64) / rot)
    angle = st["positions"].double()[..., None] * freq                     # [N, B, T, rot / 2]
    cos, sin = angle.cos().float()[..., None, :], angle.sin().float()[..., None, :]
    out = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"]) * w.float()[:, None, None, None, :]
        r, rest = y[..., :rot], y[..., rot:]
        if c["interleaved"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = r[..., :rot // 2], r[..., rot // 2:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        out.append(torch.cat((r, rest), -1).to(x.dtype))
    return tuple(out)


def _rows(st, length):
    """Page and slot of token i < length of every sequence, and which of them a sequence has: [N * B, length]."""
    page, table = st["case"]["page"], st["table"].flatten(0, 1).long()
    at = torch.arange(length, device=DEV)
    block = (at // page).clamp_max(table.shape[1] - 1)
    return table[:, block].clamp_min(0), (at % page).expand(table.shape[0], -1), at < st["lengths"].flatten()[:, None]


def _gathered(st, name, length):
    """K or V of every sequence as [N * B, length, Hkv, Dh] in fp32, zero behind its last token."""
    page, slot, has = _rows(st, length)
    x = st[name + "_pages"].transpose(1, 2)[page, slot].float()
    if st[name + "_scales"] is not None:
        x = x * st[name + "_scales"].transpose(1, 2)[page, slot][..., None]
    return torch.where(has[..., None, None], x, 0.0)


def _plain_cache(st):
    c = st["case"]
    t = torch.arange(c["t"], device=DEV)
    start, count = st["start"].flatten().long()[:, None], st["count"].flatten()[:, None]
    seq, new = torch.nonzero(t < count, as_tuple=True)
    at = start[seq, 0] + new
    page, slot = st["table"].flatten(0, 1).long()[seq, at // c["page"]], at % c["page"]
    for name in ("k", "v"):
        rows = st[name].flatten(0, 1)[seq, new]
        if c["bits"] == 8:
            rows, scales = _quantise(rows)
            st[name + "_scales"][page, :, slot] = scales
        st[name + "_pages"][page, :, slot] = rows
    if c["bits"] != 8:
        return st["k_pages"], st["v_pages"]
    shape = (c["n"], c["b"], st["max_length"], c["hkv"], c["dh"])
    return tuple(_gathered(st, name, st["max_length"]).to(DTYPES[c["dtype"]]).view(shape) for name in ("k", "v"))


def _plain_attention(st):
    c, q = st["case"], st["q"]
    n, hq, hkv, dh, length = c["n"] * c["b"], c["hq"], c["hkv"], c["dh"], c["len"]
    k = _gathered(st, "k", length).permute(0, 2, 3, 1).contiguous()        # [N * B, Hkv, Dh, length]
    s = torch.matmul(q.float().view(n, hkv, hq // hkv, dh), k) * dh ** -0.5
    del k
    has = _rows(st, length)[2]
    if st["first"] is not None:
        has = has & (torch.arange(length, device=DEV) >= st["first"].flatten()[:, None])
    s = torch.where(has[:, None, None], s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e38))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, _gathered(st, "v", length).transpose(1, 2).contiguous())
    return torch.where(total > 0, o / total, 0.0).to(q.dtype).view(q.shape)


def _plain_linear4(st):
    c, x, codes = st["case"], st["x"], st["codes"]
    w = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :c["k"]].float()
    group = torch.arange(c["k"], device=DEV) // c["group"]
    w = w - (8.0 if st["zeros"] is None else st["zeros"].float()[..., group])
    w = w * st["scales"].float()[..., group]
    return torch.matmul(x.float(), w.transpose(1, 2)).to(x.dtype)


# ---------------------------------------------------------------------------------------
# what a pass cannot do without, and how exactly it is computed
# ---------------------------------------------------------------------------------------

def work(case):
    c, es = case, 4 if case["dtype"] == "f32" else 2
    if c["kind"] == "norm":
        rows = c["n"] * c["b"] * c["t"]
        e = rows * (c["hq"] + c["hkv"]) * c["dh"]
        return {"bytes": 2 * es * e + 8 * rows + 2 * es * c["n"] * c["dh"], "flops": 8 * e}
    stored = lambda rows: 2 * rows * (c["dh"] * c["bits"] // 8 + (4 if c["bits"] == 8 else 0))  # noqa: E731
    if c["kind"] == "cache":
        rows, seqs = sum(_counts(c)) * c["hkv"], c["n"] * c["b"]
        total = 2 * rows * c["dh"] * es + stored(rows)
        if c["bits"] == 8:                              # reading back: the past tokens too, every row of the output
            back = (sum(_counts(c)) + sum(_starts(c))) * c["hkv"]
            total += stored(back) + 2 * seqs * (c["past"] + c["t"]) * c["hkv"] * c["dh"] * es
        return {"bytes": total, "flops": 4 * rows * c["dh"]}
    if c["kind"] == "attention":
        seen = sum(min(x, c["window"]) if c["window"] else x for x in _lengths(c))
        seqs = c["n"] * c["b"]
        return {"bytes": stored(seen * c["hkv"]) + 2 * seqs * c["hq"] * c["dh"] * es + 4 * seen // c["page"] + 8 * seqs,
                "flops": 4 * seen * c["hq"] * c["dh"]}
    g = -(-c["k"] // c["group"])
    return {"bytes": c["n"] * (c["o"] * ((c["k"] + 1) // 2 + g * (es + c["zeros"])) + c["m"] * (c["k"] + c["o"]) * es),
            "flops": 2 * c["n"] * c["m"] * c["o"] * c["k"]}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    with torch.no_grad():
        return {"norm": _exact_norm, "cache": _exact_cache, "attention": _exact_attention,
                "linear4": _exact_linear4}[case["kind"]](case, st)


def _exact_norm(c, st):
    """The rotation as a product of complex numbers, pair by pair."""
    half = c["rot"] // 2
    turn = torch.exp(-math.log(st["base"]) * torch.arange(half, device=DEV, dtype=torch.float64) / half)
    phase = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), st["positions"].double().unsqueeze(-1) * turn)
    first = torch.arange(half, device=DEV) * (2 if c["interleaved"] else 1)
    second = first + (1 if c["interleaved"] else half)
    res = []
    for x, w in ((st["q"], st["q_weight"]), (st["k"], st["k_weight"])):
        x = x.double()
        y = x / ((x * x).sum(-1, keepdim=True) / c["dh"] + st["eps"]).sqrt()
        y = y * w.double().view(c["n"], 1, 1, 1, c["dh"])
        z = torch.complex(y[..., first], y[..., second]) * phase.unsqueeze(3)
        y[..., first], y[..., second] = z.real, z.imag
        res.append(y)
    return tuple(res)


def _stored(x, bits):
    """What a row of the cache stands for."""
    x = x.double()
    if bits != 8:
        return x
    s = torch.clamp((x.abs().max(-1, keepdim=True).values / 127.0), min=2.0 ** -126).float().double()
    return torch.round(x / s) * s


def _value(st, name, page):
    """A page of the pool in 64 bits, [Hkv, page, Dh]."""
    x = st[name + "_pages"][page].double()
    return x if st[name + "_scales"] is None else x * st[name + "_scales"][page].double().unsqueeze(-1)


def _exact_cache(c, st):
    """Sequence by sequence."""
    table, start, count = (st[k].flatten(0, 1).tolist() for k in ("table", "start", "count"))
    out = {name: st[name + "_pages"].double() if c["bits"] != 8 else
           torch.zeros((c["n"] * c["b"], st["max_length"], c["hkv"], c["dh"]), dtype=torch.float64, device=DEV)
           for name in ("k", "v")}
    for name in ("k", "v"):
        new = st[name].flatten(0, 1)
        for i, (ids, s, t) in enumerate(zip(table, start, count)):
            used = [p for p in ids if p >= 0]
            rows = torch.cat([_value(st, name, p) for p in used], 1).transpose(0, 1).contiguous()   # [tokens, Hkv, Dh]
            rows[s:s + t] = _stored(new[i, :t], c["bits"])
            if c["bits"] == 8:
                out[name][i, :s + t] = rows[:s + t]
            else:
                for j, p in enumerate(used):
                    out[name][p] = rows[j * c["page"]:(j + 1) * c["page"]].transpose(0, 1)
    if c["bits"] != 8:
        return out["k"], out["v"]
    return tuple(out[name].view(c["n"], c["b"], *out[name].shape[1:]) for name in ("k", "v"))


def _exact_attention(c, st):
    """Sequence by sequence, over its own tokens only."""
    group = c["hq"] // c["hkv"]
    lens = st["lengths"].flatten().tolist()
    table = st["table"].flatten(0, 1)
    out = torch.zeros((len(lens), c["hq"], c["dh"]), dtype=torch.float64, device=DEV)
    q = st["q"].flatten(0, 1).double()
    for i, length in enumerate(lens):
        low = 0 if not c["window"] else max(length - c["window"], 0)
        if length <= low:
            continue
        ids = table[i, :-(-length // c["page"])].long()
        k, v = (_value(st, name, ids).transpose(0, 1).flatten(1, 2)[:, low:length] for name in ("k", "v"))
        for h in range(c["hkv"]):
            s = (q[i, h * group:(h + 1) * group] @ k[h].t().contiguous()) / math.sqrt(c["dh"])
            out[i, h * group:(h + 1) * group] = torch.softmax(s, -1) @ v[h].contiguous()
    return out.view(c["n"], c["b"], c["hq"], c["dh"])


def _exact_linear4(c, st):
    """Group by group of columns: the codes' products, scaled."""
    codes = torch.empty((c["n"], c["o"], 2 * st["codes"].shape[-1]), dtype=torch.float64, device=DEV)
    codes[..., 0::2], codes[..., 1::2] = st["codes"] % 16, st["codes"] // 16
    x = st["x"].double()
    y = torch.zeros((c["n"], c["m"], c["o"]), dtype=torch.float64, device=DEV)
    for g in range(st["scales"].shape[-1]):
        lo, hi = g * c["group"], min((g + 1) * c["group"], c["k"])
        zero = 8.0 if st["zeros"] is None else st["zeros"][..., g].double().unsqueeze(-1)
        y += (x[..., lo:hi] @ (codes[..., lo:hi] - zero).transpose(1, 2).contiguous()) \
            * st["scales"][..., g].double().unsqueeze(1)
    return y
