"""The decode-step operators together (GPU): prompts through WideAttention.prompt, then tokens through
WideAttention.step, against causal attention over the whole sequence in 64 bits; and 4-bit projections, head norms,
an 8-bit cache and its attention in a row, as a step of an ensemble of decoders with shared key heads runs them."""

import pytest
import torch

from tests._serve import attend, make_table, quantise
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _turn(x, pos, base=10000.0):
    """x [n, b, t, h, d] (64 bits) turned by position, halves paired."""
    d = x.shape[-1]
    a = (pos.double()[..., None] * base ** (-2.0 * torch.arange(d // 2, device=x.device).double() / d))[..., None, :]
    u, v = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()], -1)


def _norm(x, w, eps=1e-6):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().view(w.shape[0], 1, 1, 1, -1)


@pytest.mark.parametrize("dtype,quantized", [(torch.float32, False), (torch.bfloat16, False), (torch.float32, True)])
@pytest.mark.parametrize("normed", [False, True])
def test_prompt_then_steps(normed, dtype, quantized):
    """Row t of causal attention over the whole sequence is what step t gives (an 8-bit cache: over its rows' values).
    The bars are normwise: fp32 sums 1e-5; bf16 roundings of q, k, v, weights and two outputs 2e-2; an 8-bit cache
    moves scores and values by half a step of 1/127 of a row's largest, 1.5 % of a value of unit size."""
    import wide_compiler as wc
    n, b, d, heads, total = 2, 3, 128, 4, 37
    dh = d // heads
    torch.manual_seed(1)
    mods = [torch.nn.MultiheadAttention(d, heads, batch_first=True) for _ in range(n)]
    for m in mods:
        torch.nn.init.normal_(m.in_proj_bias, 0, 0.3)
    attn = wc.WideAttention.from_modules(mods).to(DEV, dtype).eval()
    norm = None
    if normed:
        norm = wc.WideHeadNormRotary(n, dh).to(DEV, dtype)
        torch.nn.init.normal_(norm.q_weight, 1, 0.2), torch.nn.init.normal_(norm.k_weight, 1, 0.2)
    x = torch.randn(n, b, total, d, generator=gen(2)).to(DEV, dtype)
    prompt = torch.tensor([[5, 1, 20], [16, 17, 3]], dtype=torch.int32)
    table, pages = make_table(torch.full((n, b), total, dtype=torch.int32), 16, gen(3))
    table, lens = table.to(DEV), prompt.to(DEV)
    cache = wc.WidePagedCache(pages, 16, heads, dh, dtype=dtype, quantized=quantized)
    got = torch.zeros(n, b, total, d, device=DEV, dtype=dtype)
    steps = 17                                               # every sequence: its prompt, then 17 tokens
    with torch.no_grad():
        y = attn.prompt(x[:, :, :20], cache, table, lens, head_norm=norm)
        for i in range(n):
            for j in range(b):
                got[i, j, :int(prompt[i, j])] = y[i, j, :int(prompt[i, j])]
        rows, cols = torch.arange(n, device=DEV)[:, None], torch.arange(b, device=DEV)
        for _ in range(steps):
            lens = lens + 1
            at = lens.long() - 1
            got[rows, cols, at] = attn.step(x[rows, cols, at], cache, table, lens, head_norm=norm)
    cache.index_error()
    w = lambda t: t.detach().double()  # noqa: E731
    xd = x.double().reshape(n, b * total, d)
    proj = lambda wt, bias: (torch.bmm(xd, wt.transpose(1, 2).contiguous()) + bias[:, None]).view(n, b, total, heads, dh)  # noqa: E731
    q = proj(w(attn.q_weight), w(attn.q_bias))
    k = proj(w(attn.kv_weight)[:, :d], w(attn.kv_bias)[:, :d])
    v = proj(w(attn.kv_weight)[:, d:], w(attn.kv_bias)[:, d:])
    if normed:
        pos = torch.arange(total, device=DEV).expand(n, b, total)
        q, k = _turn(_norm(q, norm.q_weight), pos), _turn(_norm(k, norm.k_weight), pos)
    ref = torch.zeros(n, b, total, d, device=DEV, dtype=torch.float64)
    kq, vq = (quantise(k), quantise(v)) if quantized else (k, v)
    for t in range(total):
        one = torch.full((n, b), t + 1, device=DEV, dtype=torch.int32)
        o, _ = attend(q[:, :, t], k[:, :, :t + 1], v[:, :, :t + 1], one)
        if quantized:                                        # tokens after the prompt attend over the cache
            oq, _ = attend(q[:, :, t], kq[:, :, :t + 1], vq[:, :, :t + 1], one)
            o = torch.where((t >= prompt.to(DEV))[..., None, None], oq, o)
        ref[:, :, t] = torch.einsum("nbd,nod->nbo", o.flatten(-2), w(attn.out_weight)) + w(attn.out_bias)[:, None]
    seen = torch.arange(total, device=DEV) < (prompt.to(DEV) + steps)[..., None]
    # fp32 keys next to a code's border may round the other way: one code of 127 in a value
    bar = 2e-2 if dtype == torch.bfloat16 else 1e-3 if quantized else 1e-5
    err = ((got.double() - ref)[seen].abs().max() / ref[seen].abs().max()).item()
    assert err <= bar, err


def test_inactive_sequences_take_no_part():
    import wide_compiler as wc
    attn = wc.WideAttention(2, 64, 2).to(DEV).eval()
    cache = wc.WidePagedCache(4, 8, 2, 32, dtype=torch.float32)
    table = torch.tensor([[[0], [-1]], [[2], [3]]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([[1, 0], [1, 1]], dtype=torch.int32, device=DEV)
    x = torch.randn(2, 2, 64, device=DEV)
    with torch.no_grad():
        y = attn.step(x, cache, table, lens)
    cache.index_error()
    assert torch.equal(y[0, 1], attn.out_bias[0]) and (cache.k_pages[1] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_decoder_step_with_shared_heads(dtype):
    """x -> 4-bit q|k|v -> head norms with rotation -> 8-bit cache -> attention -> 4-bit output, captured as a graph and
    replayed token by token against the same chain in 64 bits, which rounds where tensors of the type lie between.
    Bar: 8 roundings of half a step on the way, and one code in 254 of the largest of a row of k and of v."""
    import wide_compiler as wc
    n, b, hq, hk, dh, page, d = 2, 3, 8, 2, 64, 8, 256
    g = gen(5)
    lin = lambda i, o: [torch.nn.Linear(i, o).to(DEV, dtype) for _ in range(n)]  # noqa: E731
    torch.manual_seed(6)
    qkv = wc.WideLinear4bit.from_modules(lin(d, (hq + 2 * hk) * dh), 64)
    out = wc.WideLinear4bit.from_modules(lin(hq * dh, d), 64)
    norm = wc.WideHeadNormRotary(n, dh).to(DEV, dtype)
    total = 20
    table, pages = make_table(torch.full((n, b), total, dtype=torch.int32), page, g)
    table = table.to(DEV)
    cache = wc.WidePagedCache(pages, page, hk, dh, dtype=dtype, quantized=True)
    x = torch.randn(n, b, 1, d, generator=g).to(DEV, dtype)
    start = torch.tensor([[0, 0, 0], [0, -1, 0]], dtype=torch.int32, device=DEV)
    lens = start + 1

    def step():
        h = qkv(x)
        q, k = norm(h[..., :hq * dh].unflatten(-1, (hq, dh)), h[..., hq * dh:(hq + hk) * dh].unflatten(-1, (hk, dh)),
                    start[..., None])
        cache.write(k, h[..., (hq + hk) * dh:].unflatten(-1, (hk, dh)), table, start)
        return out(cache.attend(q[:, :, 0], table, lens).flatten(-2))

    ks, vs = [], []
    wq, wo = qkv.dequantize().double(), out.dequantize().double()
    with torch.no_grad():
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
        half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11
        for t in range(total):
            x.copy_(torch.randn(n, b, 1, d, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            h = (torch.bmm(x.double()[:, :, 0], wq.transpose(1, 2).contiguous()) + qkv.bias.double()[:, None])[:, :, None].to(dtype)
            heads = lambda lo, hi: h[..., lo * dh:hi * dh].unflatten(-1, (hi - lo, dh))  # noqa: E731
            pos = start[..., None]
            ks.append(quantise(_turn(_norm(heads(hq, hq + hk), norm.k_weight), pos).to(dtype)))
            vs.append(quantise(heads(hq + hk, hq + 2 * hk)))
            q = _turn(_norm(heads(0, hq), norm.q_weight), pos).to(dtype)
            o, _ = attend(q[:, :, 0], torch.cat(ks, 2), torch.cat(vs, 2), lens)
            ref = torch.bmm(o.to(dtype).double().flatten(-2), wo.transpose(1, 2).contiguous()) + out.bias.double()[:, None]
            err = ((y.double() - ref)[:, [0, 2]].abs().max() / ref.abs().max()).item()
            assert err <= 8 * half + 1 / 254, (t, err)
            assert torch.equal(y[1, 1], out.bias[1])
            start.add_((start >= 0).to(torch.int32))
            lens.copy_(start + 1)
    cache.index_error()


def test_a_refused_prompt_leaves_the_cache():
    import wide_compiler as wc
    attn = wc.WideAttention(2, 256, 1).to(DEV).eval()
    cache = wc.WidePagedCache(8, 16, 1, 256, dtype=torch.float32)
    table = torch.arange(2, dtype=torch.int32, device=DEV).view(2, 1, 1)
    lens = torch.full((2, 1), 5, dtype=torch.int32, device=DEV)
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="256 columns"):
            attn.prompt(torch.randn(2, 1, 5, 256, device=DEV), cache, table, lens)
        assert (cache.k_pages == 0).all()
        assert torch.isfinite(attn.step(torch.randn(2, 1, 256, device=DEV), cache, table, lens)).all()


def test_under_torch_compile():
    """A compiled function ends its regions at these calls, and gives what the function itself gives."""
    import wide_compiler as wc
    n, b, h, d = 2, 3, 2, 64
    attn = wc.WideAttention(n, h * d, h).to(DEV, torch.bfloat16).eval()
    norm = wc.WideHeadNormRotary(n, d).to(DEV, torch.bfloat16)
    proj = wc.WideLinear4bit.from_modules([torch.nn.Linear(h * d, 40).to(DEV, torch.bfloat16) for _ in range(n)], group_size=32)
    lens = torch.tensor([[5, 1, 0], [9, 30, 2]], dtype=torch.int32)
    table, pages = make_table(lens, 16, gen(3))
    table, lens = table.to(DEV), lens.to(DEV)
    x = torch.randn(n, b, h * d, device=DEV, dtype=torch.bfloat16)
    outs = []
    for wrap in (lambda f: f, lambda f: torch.compile(f, backend="eager")):
        cache = wc.WidePagedCache(pages, 16, h, d)

        def step(x, table, lens):
            y = attn.step(x, cache, table, lens, norm)
            k, v = cache.read(table, lens, 30)
            return proj(y + 1), k, v
        with torch.no_grad():
            outs.append(wrap(step)(x, table, lens))
    for a, c in zip(*outs):
        assert torch.equal(a, c)
