"""The operators that draw many answers to the same prompts, together (GPU): prompts through WideAttention.prompt, then the
answers' tokens through WideAttention.step over the shared prefixes, against causal attention over each whole sequence
in 64 bits; and a decoder of 8-bit projections, shared prefixes and a sampler, whose tokens go back in, as a captured graph."""

import pytest
import torch

from tests._answer import draw, linear8, shared
from tests._serve import attend, attend_slack, make_table, quantise, within
from tests._util import gen
from tests.test_gpu_decode import _norm, _turn

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("dtype,quantized", [(torch.float32, False), (torch.bfloat16, False), (torch.float32, True)])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("share", [3, 20])
def test_prompts_then_steps_of_many_answers(share, normed, dtype, quantized):
    """Step t of an answer is row prefix + t of causal attention over its prompt and its tokens.  Bars, normwise: fp32 sums
    1e-5; bf16 roundings of q, k, v, weights and two outputs 2e-2; codes next to a border of an 8-bit cache 1e-3."""
    import wide_compiler as wc
    n, groups, d, heads, steps = 2, 2, 64, 2, 6
    dh, b = d // heads, groups * share
    torch.manual_seed(1)
    mods = [torch.nn.MultiheadAttention(d, heads, batch_first=True) for _ in range(n)]
    attn = wc.WideAttention.from_modules(mods).to(DEV, dtype).eval()
    norm = wc.WideHeadNormRotary(n, dh).to(DEV, dtype) if normed else None
    lengths = torch.tensor([[70, 0], [33, 16]], dtype=torch.int32)
    x = torch.randn(n, groups, 70, d, generator=gen(2)).to(DEV, dtype)
    new = torch.randn(n, b, steps, d, generator=gen(3)).to(DEV, dtype)
    table, p0 = make_table(lengths, 16, gen(4))
    own, p1 = make_table(torch.full((n, b), steps, dtype=torch.int32), 16, gen(5))
    own = (own + p0)[..., :1]
    active = (torch.arange(b) % 5 != 4).expand(n, b)
    cache = wc.WidePagedCache(p0 + p1, 16, heads, dh, dtype=dtype, quantized=quantized)
    table, own, common = table.to(DEV), own.contiguous().to(DEV), lengths.to(DEV)
    got = []
    with torch.no_grad():
        attn.prompt(x, cache, table, common, head_norm=norm)
        for t in range(steps):
            lens = torch.where(active, t + 1, 0).int().to(DEV)
            got.append(attn.step(new[:, :, t], cache, own, lens, head_norm=norm, prefix=(table, common)))
    cache.index_error()
    w = lambda t: t.detach().double()  # noqa: E731
    wide = torch.cat([x.double().repeat_interleave(share, 1), torch.zeros_like(new).double()], 2)      # a prompt, then its answer
    start = lengths.repeat_interleave(share, 1)
    for i in range(n):
        for j in range(b):
            wide[i, j, start[i, j]:start[i, j] + steps] = new[i, j].double()
    total = wide.shape[2]
    flat = wide.reshape(n, b * total, d)
    proj = lambda wt, bias: (torch.bmm(flat, wt.transpose(1, 2).contiguous()) + bias[:, None]).view(n, b, total, heads, dh)  # noqa: E731
    q = proj(w(attn.q_weight), w(attn.q_bias))
    k = proj(w(attn.kv_weight)[:, :d], w(attn.kv_bias)[:, :d])
    v = proj(w(attn.kv_weight)[:, d:], w(attn.kv_bias)[:, d:])
    if normed:
        pos = torch.arange(total, device=DEV).expand(n, b, total)
        q, k = _turn(_norm(q, norm.q_weight), pos), _turn(_norm(k, norm.k_weight), pos)
    if quantized:
        k, v = quantise(k), quantise(v)
    bar = 2e-2 if dtype == torch.bfloat16 else 1e-3 if quantized else 1e-5
    rows, cols = torch.arange(n, device=DEV)[:, None], torch.arange(b, device=DEV)
    for t in range(steps):
        at = (start + t).long().to(DEV)
        o, _ = attend(q[rows, cols, at], k, v, (at + 1).int())
        ref = torch.bmm(o.flatten(-2), w(attn.out_weight).transpose(1, 2).contiguous()) + w(attn.out_bias)[:, None]
        err = ((got[t].double() - ref)[active.to(DEV)].abs().max() / ref.abs().max()).item()
        assert err <= bar, (t, err)
        none = w(attn.out_bias).to(dtype)[:, None].expand(n, b, d)
        assert torch.equal(got[t][~active.to(DEV)], none[~active.to(DEV)])          # a place without an answer takes no part


def test_refusals_of_a_prefix():
    import wide_compiler as wc
    attn = wc.WideAttention(1, 64, 2).to(DEV).eval()
    cache = wc.WidePagedCache(4, 8, 2, 32, dtype=torch.float32)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    x = torch.zeros(1, 4, 64, device=DEV)
    with torch.no_grad():
        for common in (i(1, 3), i(2, 2), i(2), i(1, 0)):
            with pytest.raises(RuntimeError, match="WideAttention.step"):
                attn.step(x, cache, i(1, 4, 1), i(1, 4), prefix=(i(1, 2, 1), common))


@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, False)])
def test_a_decoder_draws_answers(dtype, quantized):
    """tokens -> embedding -> 8-bit q|k|v -> head norms -> cache -> attention over shared prefixes -> 8-bit output ->
    8-bit logits -> sampler -> tokens, captured as a graph and replayed token by token.  Each replay gives what the same
    calls one by one give, bit for bit, on a cache of their own; and each operator its plain form of what went into it."""
    import wide_compiler as wc
    n, groups, share, hq, hk, dh, page, d, vocab, prompt, steps = 2, 2, 6, 8, 2, 64, 8, 128, 1003, 45, 5
    b, g = groups * share, gen(7)
    torch.manual_seed(8)
    lin = lambda i, o: wc.WideLinear8bit.from_modules([torch.nn.Linear(i, o).to(DEV, dtype) for _ in range(n)])  # noqa: E731
    qkv, out, head = lin(d, (hq + 2 * hk) * dh), lin(hq * dh, d), lin(d, vocab)
    embed = wc.WideEmbedding.from_modules([torch.nn.Embedding(vocab, d) for _ in range(n)]).to(DEV, dtype)
    norm = wc.WideHeadNormRotary(n, dh).to(DEV, dtype)
    sampler = wc.WideSampler(n, temperature=[0.8, 1.1], top_k=[0, 40], top_p=[0.9, 1.0], min_p=[0.0, 0.02]).to(DEV)
    common = torch.tensor([[prompt, 17], [1, prompt]], dtype=torch.int32)
    table, p0 = make_table(common, page, g)
    own, p1 = make_table(torch.full((n, b), steps, dtype=torch.int32), page, g)
    own = torch.where(own >= 0, own + p0, own).to(DEV)
    table, common = table.to(DEV), common.to(DEV)
    keys, values = (torch.randn(n, groups, prompt, hk, dh, generator=g).to(DEV, dtype) for _ in range(2))
    active = torch.ones(n, b, dtype=torch.bool, device=DEV)
    active[0, 3], active[1, 11] = False, False
    none = torch.zeros(n, groups, dtype=torch.int32, device=DEV)

    def state():
        cache = wc.WidePagedCache(p0 + p1, page, hk, dh, dtype=dtype, quantized=quantized)
        cache.write(keys, values, table, none, common)
        return cache, torch.zeros(n, b, dtype=torch.int64, device=DEV), torch.zeros(n, b, dtype=torch.int32, device=DEV), \
            torch.zeros(n, b, device=DEV)

    def step(cache, tokens, start, u):
        x = embed(tokens, per_model=True)
        h = qkv(x)
        at = (start + common.repeat_interleave(share, 1))[..., None]
        q, k = norm(h[:, :, None, :hq * dh].unflatten(-1, (hq, dh)), h[:, :, None, hq * dh:(hq + hk) * dh].unflatten(-1, (hk, dh)), at)
        cache.write(k, h[:, :, None, (hq + hk) * dh:].unflatten(-1, (hk, dh)), own, torch.where(active, start, -1))
        lens = torch.where(active, start + 1, -1)
        o = cache.attend_shared(q[:, :, 0], table, common, own, lens)
        y = out(o.flatten(-2))
        logits = head(x + y)
        drawn = sampler(logits, u)
        tokens.copy_(drawn.clamp_min(0))
        start.add_(1)
        return x, h, q[:, :, 0], lens, o, y, logits, drawn

    half = HALF[dtype]
    with torch.no_grad():
        captured, eager = state(), state()
        step(*state())                                       # workspaces and plans, on a state that is not used
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            seen = step(*captured)
        for t in range(steps):
            u = torch.rand(n, b, generator=g).to(DEV)
            captured[3].copy_(u), eager[3].copy_(u)
            graph.replay()
            torch.cuda.synchronize()
            plain = step(*eager)
            for a, c in zip(seen, plain):
                assert torch.equal(a, c), t
            x, h, q, lens, o, y, logits, drawn = seen
            cache = captured[0]
            pools = [p[..., :dh].double() for p in (cache.k_pages, cache.v_pages)]
            if quantized:
                pools = [p * s.double()[..., None] for p, s in zip(pools, (cache.k_scales, cache.v_scales))]
            ref, big = shared(q, *pools, table, common, own, lens)
            bars = attend_slack(dtype, big, dh, prompt + steps, pools[1].abs().max().item())
            within(o, ref, half + 2.0 ** -23, bars)
            # a product: its two scales, their product and the sum with the bias in fp32, then the result
            for mod, i, r in ((qkv, x, h), (out, o.flatten(-2), y), (head, x + y, logits)):
                codes = torch.round(mod.dequantize().double() / mod.scales.double()[..., None])
                alone, full = linear8(i, codes, mod.scales, mod.bias)
                within(r, full, half + 2 * 2.0 ** -24, 4 * 2.0 ** -24 * alone.abs())
            rules = [(0.8, 0, 0.9, 0.0), (1.1, 40, 1.0, 0.02)]
            assert drawn.tolist() == [[draw(logits[i, j], u[i, j].item(), *rules[i]) for j in range(b)] for i in range(n)]
            assert (o[~active] == 0).all()
    cache.index_error()
    assert (captured[2] == steps).all()


def test_under_torch_compile():
    """A compiled function ends its regions at these calls, and gives what the function itself gives."""
    import wide_compiler as wc
    n, b, h, d = 2, 4, 2, 64
    attn = wc.WideAttention(n, h * d, h).to(DEV, torch.bfloat16).eval()
    head = wc.WideLinear8bit.from_modules([torch.nn.Linear(h * d, 40).to(DEV, torch.bfloat16) for _ in range(n)])
    sampler = wc.WideSampler(n, top_p=0.9).to(DEV)
    common = torch.tensor([[20, 0], [1, 9]], dtype=torch.int32)
    table, p0 = make_table(common, 8, gen(1))
    own, p1 = make_table(torch.full((n, b), 3, dtype=torch.int32), 8, gen(2))
    table, common, own = table.to(DEV), common.to(DEV), (own + p0).to(DEV)
    kv = torch.randn(n, 2, 20, h, d, device=DEV, dtype=torch.bfloat16)
    x, u = torch.randn(n, b, h * d, device=DEV, dtype=torch.bfloat16), torch.rand(n, b, device=DEV)
    lens = torch.tensor([[1, 3, 0, 2], [2, 1, 1, 3]], dtype=torch.int32, device=DEV)
    outs = []
    for wrap in (lambda f: f, lambda f: torch.compile(f, backend="eager")):
        cache = wc.WidePagedCache(p0 + p1, 8, h, d)
        cache.write(kv, kv, table, torch.zeros_like(common), common)

        def step(x, lens, u):
            y = attn.step(x, cache, own, lens, prefix=(table, common))
            logits = head(y + 1)
            return y, logits, sampler(logits, u), cache.attend_shared(x.view(n, b, h, d), table, common, own, lens)
        with torch.no_grad():
            outs.append(wrap(step)(x, lens, u))
    for a, c in zip(*outs):
        assert torch.equal(a, c)
