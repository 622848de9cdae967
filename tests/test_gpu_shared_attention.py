"""Attention over shared prefixes and own tokens (GPU) against softmax over both in 64 bits."""

import pytest
import torch

from tests._answer import shared
from tests._serve import HALF, attend_slack, make_table, quantise, within
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _make(prefix, lens, hq, hkv, dh, page, dtype, bits, seed=0):
    """A cache whose unused slots hold NaN, its values, tables and queries."""
    import wide_compiler as wc
    g = gen(seed)
    prefix, lens = torch.tensor(prefix, dtype=torch.int32), torch.tensor(lens, dtype=torch.int32)
    pt, p0 = make_table(prefix.clamp_min(0), page, g)
    table, p1 = make_table(lens.clamp_min(0), page, g)
    table = torch.where(table >= 0, table + p0, table)
    cache = wc.WidePagedCache(p0 + p1, page, hkv, dh, dtype=dtype, quantized=bits == 8)
    n = lens.shape[0]
    for t, l in ((pt, prefix), (table, lens)):
        most = max(int(l.max()), 1)
        k, v = (torch.randn(n, l.shape[1], most, hkv, dh, generator=g).to(DEV, dtype) for _ in range(2))
        cache.write(k, v, t.to(DEV), torch.zeros_like(l).to(DEV), l.clamp_min(0).to(DEV))
    cache.index_error()
    used = torch.zeros(p0 + p1, page, dtype=torch.bool)
    for t, l in ((pt, prefix), (table, lens)):
        for i in range(n):
            for j in range(l.shape[1]):
                for x in range(max(int(l[i, j]), 0)):
                    used[t[i, j, x // page], x % page] = True
    free = ~used.to(DEV)[:, None, :].expand(-1, hkv, -1)
    for pool in ((cache.k_scales, cache.v_scales) if bits == 8 else (cache.k_pages, cache.v_pages)):
        pool[free] = float("nan")
    q = torch.randn(n, lens.shape[1], hq, dh, generator=g).to(DEV, dtype)
    return cache, q, pt.to(DEV), prefix.to(DEV), table.to(DEV), lens.to(DEV)


def _values(cache):
    if not cache.quantized:
        return cache.k_pages[..., :cache.head_dim].double(), cache.v_pages[..., :cache.head_dim].double()
    return tuple((c[..., :cache.head_dim].double() * s.double()[..., None]) for c, s in
                 ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)))


def _bars(cache, big, total, planes=2.0 ** -16):
    k, v = _values(cache)
    return attend_slack(cache.dtype, big, cache.head_dim, total, v.nan_to_num(0).abs().max().item(), planes)


def _planes(cache, q, prefix, lens):
    """What of a weight is left out.  In 16 bits, over prefixes of more than 32 rows a key head, heads of up to 128 columns,
    weights are rounded to the type once (over 8-bit pages bf16's, in fp16 two of them): half a step of each, so at most that of
    the largest value in a sum whose weights add up to one."""
    rows = lens.shape[1] // max(prefix.shape[1], 1) * (q.shape[2] // cache.n_kv_heads)
    if cache.dtype == torch.float32 or rows <= 32 or cache.head_dim > 128 or (cache.quantized and cache.dtype == torch.float16):
        return 2.0 ** -16
    return HALF[cache.dtype]


def _check(made, **kw):
    cache, q, pt, prefix, table, lens = made
    planes = _planes(cache, q, prefix, lens)
    with torch.no_grad():
        o = cache.attend_shared(q, pt, prefix, table, lens, **kw)
    cache.index_error()
    ref, big = shared(q, *_values(cache), pt, prefix, table, lens, scale=kw.get("scale"))
    total = int(prefix.max()) + max(int(lens.max()), 0)
    within(o, ref, HALF[cache.dtype] + 2.0 ** -23, _bars(cache, big, total, planes))
    return o


# (prefix lengths, own lengths, query heads, key heads): one row to a key head, several tiles of rows and ragged ones; tokens that
# end inside a tile, a page and at their ends; sequences without tokens of their own, places without a sequence
SHAPES = [
    ([[1]], [[1]], 1, 1), ([[0]], [[3]], 2, 1), ([[5]], [[0]], 2, 2), ([[33]], [[1, 2]], 4, 2),
    ([[100, 31]], [[1, 0, 64, 5]], 8, 2), ([[70], [64]], [[3, -1, 9], [0, 31, 32]], 6, 2),
    ([[257, 0, 90]], [[7, 0, -1, 40, 1, 100]], 5, 1), ([[300]], [list(range(17))], 1, 1), ([[130]], [[5] * 33], 2, 2),
    ([[65, 400]], [[(7 * i) % 23 - 1 for i in range(26)]], 14, 2), ([[600]], [[3] * 64], 4, 1), ([[95]], [[2] * 70], 6, 3),
]


@pytest.mark.parametrize("dh,page", [(64, 16), (128, 8), (80, 24), (32, 5)])
@pytest.mark.parametrize("dtype,bits", [(d, b) for d in DTYPES for b in (0, 8)])
def test_attends_over_both(dh, page, dtype, bits):
    for i, (prefix, lens, hq, hkv) in enumerate(SHAPES):
        _check(_make(prefix, lens, hq, hkv, dh, page, dtype, bits, seed=i))


@pytest.mark.parametrize("dh", [1, 7, 33, 96, 100, 136, 200, 256])
@pytest.mark.parametrize("dtype,bits", [(d, b) for d in DTYPES for b in (0, 8)])
def test_head_dims(dh, dtype, bits):
    for prefix, lens, hq, hkv in (SHAPES[4], SHAPES[8], SHAPES[9]):
        _check(_make(prefix, lens, hq, hkv, dh, 16, dtype, bits))


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0), (torch.float16, 0), (torch.bfloat16, 8), (torch.float32, 0)])
def test_long_ones_are_cut(dtype, bits):
    """Prefixes and own tokens over many shares, uneven ones that share a share."""
    for prefix, lens, hq, hkv in (([[5000, 40, 9]], [[1, 2000, 0, 30, 7, 1]], 4, 2), ([[20000]], [[1500, 5, -1]], 8, 1),
                                  ([[3000], [1]], [[2] * 40, [1] * 40], 4, 1)):
        _check(_make(prefix, lens, hq, hkv, 64, 16, dtype, bits))


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0), (torch.float16, 8), (torch.float32, 0)])
def test_bounds_and_scale(dtype, bits):
    made = _make([[90, 200]], [[4, 0, 17, 33]], 4, 2, 64, 16, dtype, bits)
    _check(made, max_prefix=200, max_length=33)
    _check(made, max_prefix=5000, max_length=90000, scale=0.3)
    _check(made, scale=0.0)
    _check(made, scale=-0.2)


def test_lengths_beyond_the_bounds_are_cut_and_reported():
    cache, q, pt, prefix, table, lens = _make([[90, 200]], [[4, 0, 17, 33]], 4, 2, 64, 16, torch.bfloat16, 0)
    with torch.no_grad():
        for kw, p, l in ((dict(max_prefix=100), [[90, 100]], lens.tolist()), (dict(max_length=20), prefix.tolist(), [[4, 0, 17, 20]])):
            got = cache.attend_shared(q, pt, prefix, table, lens, **kw)
            with pytest.raises(IndexError):
                cache.index_error()
            want = cache.attend_shared(q, pt, torch.tensor(p, dtype=torch.int32, device=DEV), table,
                                       torch.tensor(l, dtype=torch.int32, device=DEV))
            cache.index_error()
            assert torch.equal(got, want)


@pytest.mark.parametrize("bits", [0, 8])
def test_bad_pages_are_not_followed(bits):
    cache, q, pt, prefix, table, lens = _make([[40, 40]], [[20, 20, 20, 20]], 2, 1, 64, 16, torch.bfloat16, bits)
    bad = pt.clone()
    bad[0, 0, 1] = 1 << 30
    with torch.no_grad():
        got = cache.attend_shared(q, bad, prefix, table, lens)
        with pytest.raises(IndexError):
            cache.index_error()
        assert torch.isfinite(got).all()
        want = cache.attend_shared(q, pt, prefix, table, lens)
        assert torch.equal(got[:, 2:], want[:, 2:]) and not torch.equal(got[:, :2], want[:, :2])
        bad = table.clone()
        bad[0, 3, 0] = -7
        got = cache.attend_shared(q, pt, prefix, bad, lens)
        with pytest.raises(IndexError):
            cache.index_error()
        assert torch.equal(got[:, :3], want[:, :3])
        # a table without entries names no tokens
        got = cache.attend_shared(q, pt[..., :0], torch.zeros_like(prefix), table, lens)
        cache.index_error()
        one = cache.attend(q, table, lens)
        assert (got.float() - one.float()).abs().max() <= 2.0 ** -7 * one.abs().max()


def test_infinities_in_the_cache():
    """An infinite value takes an output to its infinity, an infinite key of the other sign leaves its token out."""
    for share in (2, 40):
        cache, q, pt, prefix, table, lens = _make([[50]], [[3] * share], 2, 1, 64, 16, torch.bfloat16, 0)
        q = q.abs()
        cache.v_pages[pt[0, 0, 0], 0, 4, 9] = float("inf")
        cache.k_pages[pt[0, 0, 1], 0, 2] = -float("inf")
        cache.v_pages[pt[0, 0, 1], 0, 2] = 7.0
        with torch.no_grad():
            o = cache.attend_shared(q, pt, prefix, table, lens)
        rest = torch.ones(64, dtype=torch.bool)
        rest[9] = False
        assert (o[..., 9] == float("inf")).all() and torch.isfinite(o[..., rest.to(DEV)]).all()


def test_queries_by_their_strides():
    cache, q, pt, prefix, table, lens = _make([[90, 31]], [[4, 0, 17, 33]], 6, 2, 64, 16, torch.bfloat16, 0)
    with torch.no_grad():
        want = cache.attend_shared(q, pt, prefix, table, lens)
        big = torch.zeros(1, 4, 3, 6, 65, device=DEV, dtype=torch.bfloat16)
        for view in (big[:, :, 1, :, 1:], big[:, :, 2, :, :64], big.transpose(1, 3)[:, :, 0, :, :64].transpose(1, 2)):
            view.copy_(q)
            assert torch.equal(cache.attend_shared(view, pt, prefix, table, lens), want)
        wide = torch.full((1, 4, 9), -1, dtype=torch.int32, device=DEV)
        wide[:, :, :table.shape[2]] = table
        assert torch.equal(cache.attend_shared(q, pt, prefix, wide[..., :table.shape[2]], lens, max_length=lens.max().item()), want)


def test_a_graph_follows_lengths_and_two_share_nothing():
    made = [_make([[100, 31]], [[1, 0, 64, 5]], 8, 2, 64, 16, torch.bfloat16, 0, seed=s) for s in (1, 2)]
    graphs = []
    with torch.no_grad():
        for cache, q, pt, prefix, table, lens in made:
            cache.attend_shared(q, pt, prefix, table, lens)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                o = cache.attend_shared(q, pt, prefix, table, lens)
            graphs.append((graph, o))
        sides = [torch.cuda.Stream(), torch.cuda.Stream()]
        for step in range(4):
            for (cache, q, pt, prefix, table, lens) in made:
                prefix.copy_(torch.tensor([[100 - 20 * step, 31 - step]], dtype=torch.int32))
                lens.copy_(torch.tensor([[1, 0, 64 - step, 5 - 2 * step]], dtype=torch.int32))
            torch.cuda.synchronize()
            for s, (graph, _) in zip(sides, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for m, (_, o) in zip(made, graphs):
                assert torch.equal(m[0].attend_shared(*m[1:]), o)


def test_nothing_to_do():
    import wide_compiler as wc
    cache = wc.WidePagedCache(4, 16, 2, 64)
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    with torch.no_grad():
        for n, g, b, h in ((0, 1, 2, 4), (1, 1, 0, 4), (1, 2, 0, 4), (1, 0, 0, 4), (1, 1, 2, 0)):
            assert cache.attend_shared(torch.zeros(n, b, h, 64, device=DEV, dtype=torch.bfloat16), i(n, g, 3), i(n, g), i(n, b, 2),
                                       i(n, b)).shape == (n, b, h, 64)
        o = cache.attend_shared(torch.ones(1, 2, 4, 64, device=DEV, dtype=torch.bfloat16), i(1, 1, 3), i(1, 1), i(1, 2, 2), i(1, 2))
        assert (o == 0).all()
        empty = wc.WidePagedCache(0, 16, 2, 64)
        assert (empty.attend_shared(torch.ones(1, 2, 4, 64, device=DEV, dtype=torch.bfloat16), i(1, 1, 3), i(1, 1) + 5, i(1, 2, 2),
                                    i(1, 2) + 3) == 0).all()


def test_equals_attention_of_each_sequence():
    """Sequences of one model whose block tables name the prefix's pages first, by attend."""
    made = _make([[64, 32]], [[9, 0, 40, 1, 3, 17]], 8, 2, 128, 16, torch.float32, 0)
    cache, q, pt, prefix, table, lens = made
    o = _check(made)
    share = 3
    for b in range(6):
        p = int(prefix[0, b // share])
        both = torch.cat([pt[0, b // share, :p // 16], table[0, b]])[None, None]
        with torch.no_grad():
            one = cache.attend(q[:, b:b + 1], both.contiguous(), lens[:, b:b + 1] + p)
        assert (one - o[:, b:b + 1]).abs().max() <= 2.0 ** -20


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0), (torch.float16, 0), (torch.bfloat16, 8), (torch.float16, 8), (torch.float32, 0)])
@pytest.mark.parametrize("rise", [0.02, 0.3, 5.0, -5.0, 12.0])
def test_scores_that_rise_along_the_tokens(rise, dtype, bits):
    """Scores that grow from the first token of a prefix to the last, by steps from a part of a weight's power of two a tile to
    many, and that fall: what is kept of earlier tokens is scaled in some tiles and not in others."""
    made = _make([[700, 333]], [[3] * 24], 8, 2, 64, 16, dtype, bits)
    cache, q, pt, prefix, table, lens = made
    g = gen(9)
    k = torch.randn(1, 2, 700, 2, 64, generator=g) * 0.1 + torch.linspace(0, rise, 700)[:, None, None]
    v = torch.randn(1, 2, 700, 2, 64, generator=g)
    cache.write(k.to(DEV, dtype), v.to(DEV, dtype), pt, torch.zeros_like(prefix), prefix)
    q.copy_((torch.randn(q.shape, generator=g) * 0.1 + 1).to(DEV, dtype))
    _check(made)


@pytest.mark.parametrize("dh", [32, 64, 80, 128])
@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0), (torch.bfloat16, 8), (torch.float16, 0), (torch.float16, 8)])
def test_weights_keep_their_bits_however_many_share_a_prefix(dtype, bits, dh):
    """From 1 query head to 256 to a key head, weights enter the products off by at most 2^-16 of themselves."""
    for prefix, lens, hq, hkv in (([[130]], [[1]], 1, 1), ([[130]], [[5] * 32], 1, 1), ([[130]], [[5] * 33], 1, 1), ([[40, 300]], [[3] * 32], 8, 2),
                                  ([[70]], [[2] * 65], 1, 1), ([[1000]], [[0] * 64], 4, 1)):
        cache, q, pt, prefix, table, lens = _make(prefix, lens, hq, hkv, dh, 16, dtype, bits)
        with torch.no_grad():
            o = cache.attend_shared(q, pt, prefix, table, lens)
        cache.index_error()
        ref, big = shared(q, *_values(cache), pt, prefix, table, lens)
        within(o, ref, HALF[dtype] + 2.0 ** -23, _bars(cache, big, int(prefix.max()) + int(lens.max())))


def test_a_row_hangs_little_on_how_many_share_its_prefix():
    """The same query among 1, 32, 33 and 70 sequences of a prefix: fp32 sums in other orders, weights off by 2^-16, and the result's own
    rounding are all that may differ."""
    cache, q, pt, prefix, table, lens = _make([[200]], [[4] * 70], 1, 1, 64, 16, torch.bfloat16, 0)
    k, v = _values(cache)
    ref, big = shared(q, k, v, pt, prefix, table, lens)
    with torch.no_grad():
        for share in (1, 32, 33, 70):
            o = cache.attend_shared(q[:, :share].contiguous(), pt, prefix, table[:, :share].contiguous(), lens[:, :share].contiguous())
            within(o, ref[:, :share], HALF[torch.bfloat16] + 2.0 ** -23, _bars(cache, big, 204))


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0), (torch.bfloat16, 8), (torch.float32, 0)])
@pytest.mark.parametrize("share", [3, 40])
def test_no_tokens_at_all(share, dtype, bits):
    """Prefixes without a token, own pages without one, and both, where the bounds allow long ones that would be cut."""
    for prefix, own in ((0, 0), (0, 9), (70, 0), (-1, -1), (70, -1)):
        made = _make([[prefix, prefix]], [[own] * 2 * share], 2, 1, 64, 16, dtype, bits)
        _check(made, max_prefix=5000, max_length=1000)
        _check(made, max_prefix=5000, max_length=200)
