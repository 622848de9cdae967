"""WidePagedCache.attend (GPU) against 64 bits: types, stored types, head dims, groups, pages that end inside a tile,
lengths around a tile, windows, empty sequences, strides, values that aren't finite, tables out of range, graphs.

Tolerance: half a rounding step of the result, and what attend_slack derives for the sums in fp32."""

import pytest
import torch

from tests._serve import HALF, attend, attend_slack, dense, make_table, quantise, within
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _setup(n, b, hq, hkv, d, page, lens, dtype, quantized, seed, spread=1.0):
    import wide_compiler as wc
    g = gen(seed)
    lens = torch.as_tensor(lens, dtype=torch.int32).view(n, b)
    table, pages = make_table(lens, page, g)
    cache = wc.WidePagedCache(pages, page, hkv, d, dtype=dtype, quantized=quantized)
    most = max(int(lens.max()), 1)
    k, v = (spread * torch.randn(n, b, most, hkv, d, generator=g).to(DEV) for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    q = torch.randn(n, b, hq, d, generator=g).to(DEV, dtype)
    # what no token has must never count: pools start as NaN
    if quantized:
        cache.k_scales.fill_(float("nan")), cache.v_scales.fill_(float("nan"))
    else:
        cache.k_pages[..., :d] = float("nan")
        cache.v_pages[..., :d] = float("nan")
    table, lens = table.to(DEV), lens.to(DEV)
    cache.write(k, v, table, torch.zeros_like(lens), lens)
    if quantized:
        k, v = quantise(k), quantise(v)
    return cache, q, k, v, table, lens


def _check(got, q, k, v, lens, first=None, scale=None):
    ref, big = attend(q, k, v, lens, first, scale)
    vmax = v.double().nan_to_num(0, 0, 0).abs().amax().item()
    within(got, ref, HALF[got.dtype], attend_slack(got.dtype, big, q.shape[-1], k.shape[2], vmax))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("hq,hkv,d,page", [
    (1, 1, 64, 16), (8, 8, 64, 24), (4, 1, 128, 16), (32, 8, 128, 32), (6, 2, 80, 8), (14, 2, 96, 64), (16, 1, 256, 16),
    (17, 1, 64, 7), (40, 2, 32, 128), (2, 2, 20, 1), (3, 1, 1, 5), (4, 2, 250, 33)])
def test_attend_layouts(hq, hkv, d, page, quantized, dtype):
    lens = [1, 31, 33, 100, 257, 0]
    cache, q, k, v, table, lens = _setup(2, 3, hq, hkv, d, page, lens, dtype, quantized, hq * 100 + d)
    got = cache.attend(q, table, lens)
    _check(got, q, k, v, lens)
    assert (got[1, 2] == 0).all()
    cache.index_error()


@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False),
                                             (torch.float32, True), (torch.float16, False), (torch.float16, True)])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 32, 63, 64, 127, 128, 129, 511, 1000, 4099])
def test_attend_lengths(length, dtype, quantized):
    cache, q, k, v, table, lens = _setup(1, 2, 8, 2, 128, 16, [length, max(length // 3, 1)], dtype, quantized, length)
    _check(cache.attend(q, table, lens), q, k, v, lens)
    _check(cache.attend(q, table, lens, max_length=length, scale=0.3), q, k, v, lens, scale=0.3)


@pytest.mark.parametrize("first", [[0, 0, 0, 0], [1, 31, 32, 33], [200, 5, 64, 300], [-7, 299, 150, 260]])
@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.float32, True)])
def test_attend_windows(first, dtype, quantized):
    """From any first token on; a window that starts at or behind the end is empty."""
    cache, q, k, v, table, lens = _setup(2, 2, 4, 2, 64, 16, [200, 300, 64, 260], dtype, quantized, 5)
    first = torch.tensor(first, dtype=torch.int32, device=DEV).view(2, 2)
    got = cache.attend(q, table, lens, first=first)
    _check(got, q, k, v, lens, first)
    assert (got[(first >= lens)] == 0).all()


def test_attend_strided_queries_and_tables():
    cache, q, k, v, table, lens = _setup(2, 3, 8, 2, 64, 16, [40, 7, 100, 64, 33, 1], torch.bfloat16, False, 9)
    wide = torch.full((2, 3, 8, 3 * 64 + 1), float("nan"), device=DEV, dtype=q.dtype)
    wide[..., 65:129] = q
    expect = cache.attend(q, table, lens)
    assert torch.equal(cache.attend(wide[..., 65:129], table, lens), expect)
    assert torch.equal(cache.attend(q.transpose(2, 3).contiguous().transpose(2, 3), table, lens), expect)
    padded = torch.full((2, 3, table.shape[2] + 5), 1 << 30, device=DEV, dtype=torch.int32)   # longer: not followed
    padded[..., :table.shape[2]] = table
    assert torch.equal(cache.attend(q, padded[..., :table.shape[2]], lens), expect)
    _check(cache.attend(q, padded, lens), q, k, v, lens)
    cache.index_error()


def test_attend_shared_prefix_pages():
    """Two sequences over the same pages."""
    cache, q, k, v, table, lens = _setup(1, 2, 4, 2, 64, 16, [80, 80], torch.bfloat16, False, 11)
    table[0, 1] = table[0, 0]
    lens[0, 1] = 50
    k[0, 1], v[0, 1] = k[0, 0], v[0, 0]
    _check(cache.attend(q, table, lens), q, k, v, lens)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_attend_values_far_apart(dtype):
    """One token takes nearly all the weight, ten thousand small ones share the rest; scores far from 0."""
    length, d = 10000, 64
    cache, q, k, v, table, lens = _setup(1, 1, 2, 1, d, 16, [length], dtype, False, 13)
    k = torch.zeros_like(k)
    q = torch.ones_like(q)
    k[..., 0] = -70.0
    k[:, :, 4321, :, 0] = 22.0
    v = v.abs()
    v[:, :, 4321] = 0
    zero = torch.zeros_like(lens)
    cache.write(k, v, table, zero)
    got = cache.attend(q, table, lens)
    ref, big = attend(q, k, v, lens)
    # the result is 10^4 exp(-11.5) of mean |v|: against itself, not the largest value (P's planes count relatively)
    rel = HALF[dtype] + attend_slack(dtype, big, d, length, 1.0)
    within(got, ref, rel, 0.0)


@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.float32, False), (torch.float16, True)])
def test_attend_not_finite(dtype, quantized):
    """A key or value that isn't finite shows as in the formula, in its own sequence only; what stands past a
    sequence's end in its last page does not."""
    n, b = 1, 4
    cache, q, k, v, table, lens = _setup(n, b, 4, 2, 64, 16, [70, 70, 70, 70], dtype, quantized, 17)
    k[0, 1, 33, 0] = float("nan")
    v[0, 2, 69, 1, 5] = float("inf")
    if quantized:
        v[0, 2, 69, 1] = float("nan")
    cache.write(k.to(dtype), v.to(dtype), table, torch.zeros_like(lens))
    _check(cache.attend(q, table, lens), q, k, v, lens)
    short = lens - 1                                        # the infinity is one past the end now
    ref, _ = attend(q, k, v, short)
    got = cache.attend(q, table, short)
    assert torch.isfinite(got[0, 2]).all() and torch.isfinite(ref[0, 2]).all()
    assert torch.isnan(got[0, 1, :2]).all() and torch.isfinite(got[0, 1, 2:]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attend_scores_of_minus_infinity(dtype):
    """Keys of score -infinity weigh nothing; where all are, the formula has no value (NaN)."""
    cache, q, k, v, table, lens = _setup(1, 2, 2, 1, 64, 16, [300, 40], dtype, False, 19)
    q = q.abs() + 0.1
    k[0, 0, :130, 0] = -float("inf")
    k[0, 1, :, 0] = -float("inf")
    cache.write(k, v, table, torch.zeros_like(lens), lens)
    got = cache.attend(q, table, lens)
    assert torch.isnan(got[0, 1]).all()
    ref, _ = attend(q[:, :1], k[:, :1, 130:], v[:, :1, 130:], lens[:, :1] - 130)
    big = 64.0
    within(got[:, :1], ref, HALF[dtype], attend_slack(dtype, big, 64, 300, v.double().abs().amax().item()))


def test_attend_tables_out_of_range_are_reported():
    cache, q, k, v, table, lens = _setup(1, 2, 4, 2, 64, 16, [100, 64], torch.bfloat16, False, 23)
    bad = table.clone()
    bad[0, 0, 2] = cache.num_pages
    bad[0, 1, 1] = -1
    got = cache.attend(q, bad, lens)
    with pytest.raises(IndexError):
        cache.index_error()
    cache.index_error()                                     # reported once
    # tokens of those pages take no part
    for i, lo in ((0, 32), (1, 16)):
        keep = [t for t in range(int(lens[0, i])) if not lo <= t < lo + 16]
        part = torch.tensor([[len(keep)]], dtype=torch.int32, device=DEV)
        ref, big = attend(q[:, i:i + 1], k[:, i:i + 1, keep], v[:, i:i + 1, keep], part)
        within(got[:, i:i + 1], ref, HALF[q.dtype], attend_slack(q.dtype, big, 64, 100, v.double().abs().amax().item()))
    # a length beyond the table, and beyond max_length
    got = cache.attend(q, table, lens + 1000)
    with pytest.raises(IndexError):
        cache.index_error()
    ref = cache.attend(q, table, torch.full_like(lens, 48))
    assert torch.equal(cache.attend(q, table, lens, max_length=48), ref)
    with pytest.raises(IndexError):
        cache.index_error()


def test_attend_no_pages_and_no_sequences():
    import wide_compiler as wc
    cache = wc.WidePagedCache(0, 16, 2, 64)
    q = torch.randn(1, 2, 4, 64, device=DEV, dtype=torch.bfloat16)
    lens = torch.tensor([[0, 5]], dtype=torch.int32, device=DEV)
    assert (cache.attend(q, torch.zeros(1, 2, 1, dtype=torch.int32, device=DEV), lens) == 0).all()
    assert (cache.attend(q, torch.zeros(1, 2, 0, dtype=torch.int32, device=DEV), lens) == 0).all()
    assert cache.attend(q[:, :0], torch.zeros(1, 0, 1, dtype=torch.int32, device=DEV), lens[:, :0]).shape == (1, 0, 4, 64)


def test_attend_graph_replays_follow_the_tables():
    """A captured call reads lengths, tables and pages as they are at each replay."""
    cache, q, k, v, table, lens = _setup(2, 2, 8, 2, 128, 16, [500, 300, 17, 64], torch.bfloat16, False, 29)
    cache.attend(q, table, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, table, lens)
    for step in range(4):
        lens.sub_(5 * step)
        if step == 2:
            table[0, 0, :2] = table[0, 0, :2].flip(0)
        graph.replay()
        eager = cache.attend(q, table, lens)
        torch.cuda.synchronize()
        same = torch.equal(out, eager)
        assert same, step
    cache.index_error()


def test_attend_on_another_stream():
    cache, q, k, v, table, lens = _setup(1, 4, 8, 2, 128, 16, [900, 300, 17, 64], torch.bfloat16, True, 31)
    expect = cache.attend(q, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cache.attend(q, table, lens)
    other = cache.attend(q, table, lens)                    # both at once: each call has its own workspace
    torch.cuda.synchronize()
    assert torch.equal(got, expect) and torch.equal(other, expect)


def test_attend_rows_beyond_four_gigabytes():
    """Pages whose byte offsets pass 32 bits."""
    import wide_compiler as wc
    page, d = 128, 256
    pages = (5 << 30) // (page * d * 2)
    cache = wc.WidePagedCache(pages, page, 1, d)
    g = gen(37)
    table = torch.tensor([[[pages - 1, 3, pages - 2]]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([[300]], dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, 1, 300, 1, d, generator=g).to(DEV, torch.bfloat16) for _ in range(2))
    q = torch.randn(1, 1, 2, d, generator=g).to(DEV, torch.bfloat16)
    cache.write(k, v, table, torch.zeros_like(lens))
    _check(cache.attend(q, table, lens), q, k, v, lens)
    rk, rv = cache.read(table, lens, 300)
    assert torch.equal(rk, k) and torch.equal(rv, v)


# long sequences are cut into parts that a second kernel joins
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("hq,hkv,d,page", [(1, 1, 64, 16), (17, 1, 80, 24), (40, 2, 32, 128), (16, 1, 256, 16), (6, 2, 128, 64),
                                           (3, 1, 1, 5), (4, 2, 250, 33)])
def test_attend_parts_layouts(hq, hkv, d, page, quantized, dtype):
    lens = [0, 2500, 1, 31, 0, 1300]
    cache, q, k, v, table, lens = _setup(2, 3, hq, hkv, d, page, lens, dtype, quantized, hq * 100 + d + 1)
    got = cache.attend(q, table, lens)
    _check(got, q, k, v, lens)
    assert (got[(lens == 0)] == 0).all()
    cache.index_error()


@pytest.mark.parametrize("first", [[0, 0, 0, 0], [2999, 1, 1400, 0], [3000, 0, 31, 5], [-9, -1, 33, 2600], [1234, 77, 1501, 4]])
@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, False)])
def test_attend_parts_windows(first, dtype, quantized):
    cache, q, k, v, table, lens = _setup(2, 2, 4, 2, 64, 16, [3000, 1, 1500, 2600], dtype, quantized, 41)
    first = torch.tensor(first, dtype=torch.int32, device=DEV).view(2, 2)
    got = cache.attend(q, table, lens, first=first)
    _check(got, q, k, v, lens, first)
    assert (got[(first >= lens)] == 0).all()


@pytest.mark.parametrize("n,b", [(1, 63), (1, 64), (5, 13), (3, 50), (2, 257)])
@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.float32, True)])
def test_attend_parts_of_many_sequences(n, b, dtype, quantized):
    """More sequences than a wave has lanes; most are short or empty, a few long, the last one as well."""
    g = gen(n * 1000 + b)
    lens = torch.randint(0, 60, (n * b,), generator=g) * (torch.rand(n * b, generator=g) < 0.6)
    lens[torch.randint(0, n * b, (4,), generator=g)] = 1400
    lens[-1] = 1100
    cache, q, k, v, table, lens = _setup(n, b, 2, 1, 32, 16, lens.tolist(), dtype, quantized, b)
    got = cache.attend(q, table, lens)
    _check(got, q, k, v, lens)
    assert (got[(lens == 0)] == 0).all()


def test_attend_many_long_sequences():
    """As many sequences as fill the machine stay whole at any length."""
    g = gen(43)
    lens = torch.randint(0, 40, (512,), generator=g)
    lens[100], lens[511] = 1200, 1100
    cache, q, k, v, table, lens = _setup(4, 128, 4, 4, 16, 16, lens.tolist(), torch.bfloat16, False, 43)
    _check(cache.attend(q, table, lens), q, k, v, lens)


def test_attend_parts_scores_of_minus_infinity():
    """A part whose keys all score -infinity weighs nothing next to one that has a score."""
    cache, q, k, v, table, lens = _setup(1, 1, 2, 1, 64, 16, [4000], torch.float32, False, 47)
    q = q.abs() + 0.1
    k[0, 0, :3000, 0] = -float("inf")
    cache.write(k, v, table, torch.zeros_like(lens), lens)
    got = cache.attend(q, table, lens)
    ref, _ = attend(q, k[:, :, 3000:], v[:, :, 3000:], lens - 3000)
    within(got, ref, HALF[torch.float32], attend_slack(torch.float32, 64.0, 64, 4000, v.double().abs().amax().item()))


def test_attend_forms_one_after_the_other():
    """The same cache under other queries, tables and lengths than those of the call before."""
    cache, q, k, v, table, lens = _setup(2, 2, 8, 2, 64, 16, [1500, 300, 17, 64], torch.bfloat16, False, 53)
    for cut in (2, 1, 2):
        for heads in (8, 2, 4):
            for most in (None, 1500, 1024):
                length = lens if most != 1024 else lens.clamp(max=1024)
                part = q[:, :cut, :heads]
                _check(cache.attend(part, table[:, :cut], length[:, :cut], max_length=most), part, k[:, :cut], v[:, :cut],
                       length[:, :cut])
    cache.index_error()


def test_attend_two_graphs_at_once():
    """Two captured calls that cut sequences into parts, replayed on two streams at the same time, with eager calls of
    other lengths between the replays: every call has a workspace of its own."""
    cache, q, k, v, table, lens = _setup(2, 2, 8, 2, 128, 16, [3000, 40, 1700, 2500], torch.bfloat16, False, 59)
    short = (lens // 2).contiguous()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for part in (lens, short):
        cache.attend(q, table, part)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.attend(q, table, part))
        graphs.append(g)
    for step in range(4):
        q.mul_(0.9)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        between = cache.attend(q, table, short)
        torch.cuda.synchronize()
        for out, part in zip(outs, (lens, short)):
            assert torch.equal(out, cache.attend(q, table, part)), step
        assert torch.equal(between, outs[1])
    _check(outs[0], q, k, v, lens)
    cache.index_error()


@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False),
                                             (torch.float16, True), (torch.float32, False), (torch.float32, True)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_attend_values_that_cancel(d, dtype, quantized):
    """Softmax weights count with all their bits: every token's values take away what those before it left over, so that
    the result is the rounding of the weights.  Scores are one product each, of at most 2, so a weight is off by 10 2^-24
    of itself (scale, product, difference and 2^x, of an exponent up to 2.9) and 2^-21 by its planes, a sum of 4 tokens by
    4 2^-24: 2^-19 of the sum of magnitudes in all."""
    import wide_compiler as wc
    n, b, heads, length = 2, 16, 4, 4
    g = gen(d)
    score = (2 * torch.rand(n, b, length, heads, generator=g) - 1).to(dtype).double()
    p = torch.softmax(score, 2)
    k = torch.zeros(n, b, length, heads, d, dtype=torch.float64)
    k[..., 0] = score
    if quantized:
        k = quantise(k)                                     # one value a row: its code is 127
        p = torch.softmax(k[..., 0], 2)
    v, left = [], torch.zeros(n, b, heads, d, dtype=torch.float64)
    for t in range(length):
        x = 1 + torch.rand(n, b, heads, d, generator=g, dtype=torch.float64) if t == 0 else -left / p[:, :, t, :, None]
        x = x.to(dtype)
        v.append(x)
        left = left + p[:, :, t, :, None] * (quantise(x) if quantized else x.double())
    v = torch.stack(v, 2)
    stored = quantise(v) if quantized else v.double()
    size = (p[..., None] * stored.abs()).sum(2)
    assert (left.abs() < 2.0 ** -13 * size).all()
    lens = torch.full((n, b), length, dtype=torch.int32)
    table, pages = make_table(lens, 16, g)
    cache = wc.WidePagedCache(pages, 16, heads, d, dtype=dtype, quantized=quantized)
    table, lens = table.to(DEV), lens.to(DEV)
    cache.write((score[..., None] * (torch.arange(d) == 0)).to(DEV, dtype), v.to(DEV), table, torch.zeros_like(lens))
    q = torch.zeros(n, b, heads, d, device=DEV, dtype=dtype)
    q[..., 0] = 1
    got = cache.attend(q, table, lens, scale=1.0).cpu()
    within(got, left, HALF[dtype], 2.0 ** -19 * size)


def test_attend_lengths_out_of_range_of_sequences_without_a_tile():
    """A length beyond its bound is reported in either form, also where none of the sequence's tokens is left: a pool
    without pages, a first token at or behind the bound, alone and next to sequences that have tokens."""
    import wide_compiler as wc
    for blocks in (1, 200):                                 # whole, in parts
        cache = wc.WidePagedCache(0, 16, 2, 64)
        q = torch.randn(1, 2, 4, 64, device=DEV, dtype=torch.bfloat16)
        table = torch.zeros(1, 2, blocks, dtype=torch.int32, device=DEV)
        for lens, bad in (([0, 0], False), ([0, 5], True), ([3, 0], True)):
            assert (cache.attend(q, table, torch.tensor([lens], dtype=torch.int32, device=DEV)) == 0).all()
            if bad:
                with pytest.raises(IndexError):
                    cache.index_error()
            cache.index_error()
    for most, lens in ((1000, [40, 1001, 30]), (2000, [1500, 2001, 1700])):
        cache, q, k, v, table, lens = _setup(1, 3, 4, 2, 64, 16, lens, torch.bfloat16, False, most)
        for first in ([0, most, 0], [3000, most, 3000]):
            first = torch.tensor([first], dtype=torch.int32, device=DEV)
            got = cache.attend(q, table, lens, first=first, max_length=most)
            with pytest.raises(IndexError):
                cache.index_error()
            cut = lens.clamp(max=most)
            assert torch.equal(got, cache.attend(q, table, cut, first=first, max_length=most))
            cache.index_error()


@pytest.mark.parametrize("n,b,blocks", [(1, 3, 100), (8, 8, 70), (4, 512, 70)])
def test_attend_lengths_far_beyond_the_table(n, b, blocks):
    """Lengths that say anything, under a max_length far over what the tables name: every sequence has the tokens of its
    table, and the flag is raised; in parts, and of so many sequences that they stay whole."""
    page, d = 16, 32
    full = [blocks * page] + [0] * (n * b - 1)
    cache, q, k, v, table, lens = _setup(n, b, 1, 1, d, page, full, torch.bfloat16, False, blocks)
    table[:] = table[0, 0]                                  # all of them over the same pages
    lens[:] = blocks * page
    expect = cache.attend(q, table, lens)
    cache.index_error()
    for length in (2 ** 31 - 1, 2 ** 31 - 65, blocks * page + 1):
        got = cache.attend(q, table, torch.full_like(lens, length), max_length=2 ** 31 - 65)
        with pytest.raises(IndexError):
            cache.index_error()
        within(got, expect.double(), 2 * HALF[q.dtype], attend_slack(q.dtype, 32.0, d, blocks * page, 4.5))


@pytest.mark.parametrize("dtype,quantized", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float16, False), (torch.float32, False)])
@pytest.mark.parametrize("hq,hkv,d,lens", [
    (8, 8, 64, [20000, 60000, 3000]),                       # shares of many tiles, of one sequence and of two
    (4, 1, 64, [131072]), (2, 1, 128, [300000, 17]),        # hundreds of parts, so that a thread of the join has several
    (1, 1, 32, [300000]), (16, 2, 256, [40000, 1, 9000])])
def test_attend_long_shares_and_many_parts(hq, hkv, d, lens, dtype, quantized):
    """A part adds up at most 256 products in a chain (a share's tiles over its waves, 32 tokens at a time), the join at
    most 1024 / 4 outputs: 512 additions of 2^-24 of the sum of |p v|, in numerator and sum each; a score and its
    exponential as attend_slack has them."""
    cache, q, k, v, table, lens = _setup(1, len(lens), hq, hkv, d, 64, lens, dtype, quantized, d + hq)
    got = cache.attend(q, table, lens)
    for i in range(lens.shape[1]):
        length = int(lens[0, i])
        one, part = lens[:, i:i + 1], [t[:, i:i + 1, :length] for t in (k, v)]
        ref, big = attend(q[:, i:i + 1], *part, one)
        size, _ = attend(q[:, i:i + 1], part[0], part[1].abs(), one)
        within(got[:, i:i + 1], ref, HALF[dtype], size * (2 * (d + 4) * 2.0 ** -24 * big + 2.0 ** -20 + 2 * 512 * 2.0 ** -24 + 2.0 ** -21))
    cache.index_error()
