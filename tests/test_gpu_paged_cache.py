"""WidePagedCache.write and read (GPU): what is stored in the tensors' type comes back bit for bit, 8-bit rows equal
the definition's codes and scales exactly (quotients next to a half among them) and read back as their product rounded
once; ragged counts, offsets, pages of any size, strides, padding, rows that aren't finite, tables out of range."""

import pytest
import torch

from tests._serve import dense, make_table, quantise
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _write(dtype, quantized, n, b, t, h, d, page, past, seed, scale=1.0):
    import wide_compiler as wc
    g = gen(seed)
    count = torch.randint(0, t + 1, (n, b), generator=g).to(torch.int32)
    count[0, 0] = t
    start = torch.randint(0, past + 1, (n, b), generator=g).to(torch.int32)
    table, pages = make_table(start + count, page, g)
    cache = wc.WidePagedCache(pages, page, h, d, dtype=dtype, quantized=quantized)
    k, v = ((scale * torch.randn(n, b, t, h, d, generator=g)).to(DEV, dtype) for _ in range(2))
    return cache, k, v, table.to(DEV), start.to(DEV), count.to(DEV)


def _expect(old, x, table, start, count, page, d):
    """The pool after the write, row by row: old [P, h, page, d], x [n, b, t, h, d]."""
    new = old.clone()
    for i in range(x.shape[0]):
        for j in range(x.shape[1]):
            c = int(count[i, j])
            at = int(start[i, j]) + torch.arange(c, device=x.device)
            ids = table[i, j].long()[at // page]
            new[ids, :, at % page] = x[i, j, :c].to(new.dtype)
    return new


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,b,t,h,d,page,past", [
    (1, 1, 1, 1, 64, 16, 0), (2, 3, 1, 8, 128, 16, 50), (2, 2, 70, 3, 80, 24, 100), (1, 4, 33, 2, 20, 1, 9),
    (2, 1, 130, 1, 256, 128, 300), (1, 2, 19, 5, 1, 7, 3), (3, 1, 5, 2, 250, 32, 40)])
def test_native_rows_come_back_bit_for_bit(n, b, t, h, d, page, past, dtype):
    cache, k, v, table, start, count = _write(dtype, False, n, b, t, h, d, page, past, t + d)
    cache.k_pages[..., :d] = 7.0
    cache.v_pages[..., :d] = 9.0
    before = cache.k_pages[..., :d].clone(), cache.v_pages[..., :d].clone()
    cache.write(k, v, table, start, count)
    assert torch.equal(cache.k_pages[..., :d], _expect(before[0], k, table, start, count, page, d))
    assert torch.equal(cache.v_pages[..., :d], _expect(before[1], v, table, start, count, page, d))
    assert (cache.k_pages[..., d:] == 0).all()
    lens = start + count
    most = int(lens.max()) + 3
    rk, rv = cache.read(table, lens, most)
    assert torch.equal(rk, dense(cache.k_pages[..., :d], table, lens, most))
    assert torch.equal(rv, dense(cache.v_pages[..., :d], table, lens, most))
    cache.index_error()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,b,t,h,d,page,scale", [
    (1, 1, 1, 1, 64, 16, 1.0), (2, 3, 40, 8, 128, 16, 3.0), (2, 2, 70, 3, 80, 24, 1e-3), (1, 2, 33, 2, 20, 3, 1.0),
    (2, 1, 50, 1, 256, 64, 20.0), (1, 2, 19, 5, 1, 7, 1.0)])
def test_eight_bit_rows_equal_the_definition(n, b, t, h, d, page, scale, dtype):
    cache, k, v, table, start, count = _write(dtype, True, n, b, t, h, d, page, 30, t + d, scale)
    cache.write(k, v, table, start, count)
    lens = start + count
    most = int(lens.max())
    for pages, scales, x in ((cache.k_pages, cache.k_scales, k), (cache.v_pages, cache.v_scales, v)):
        got = dense(pages.double() * scales.double()[..., None], table, lens, most)[..., :d]
        for i in range(n):
            for j in range(b):
                s, c = int(start[i, j]), int(count[i, j])
                assert torch.equal(got[i, j, s:s + c], quantise(x[i, j, :c]))
        assert (pages[..., d:] == 0).all()
    rk, _ = cache.read(table, lens, most)
    ref = dense((cache.k_pages.float() * cache.k_scales[..., None]).to(dtype), table, lens, most)[..., :d]
    assert torch.equal(rk, ref) and rk.dtype == dtype


@pytest.mark.parametrize("exponent", [-130, -126, -100, 0, 100])
def test_eight_bit_codes_next_to_a_half(exponent):
    """fp32 values at (c + 1/2) scale and one step to each side, for many scales: the nearest code, ties to even."""
    import wide_compiler as wc
    g = gen(41)
    d, rows = 128, 512
    top = (1 + torch.rand(rows, 1, generator=g, dtype=torch.float64)) * 2.0 ** exponent
    top = top.float()
    s = (top.double() / 127).clamp_min(2.0 ** -126).float()
    c = torch.arange(-21, 21, dtype=torch.float64) * 3
    mid = ((c + 0.5) * s.double()).float()
    x = torch.cat([top, mid, torch.nextafter(mid, torch.tensor(torch.inf)), torch.nextafter(mid, torch.tensor(-torch.inf))], 1)
    x = torch.cat([x, torch.zeros(rows, d - x.shape[1])], 1)
    x = torch.where(x.abs() <= top, x, top)
    cache = wc.WidePagedCache(rows // 16, 16, 1, d, dtype=torch.float32, quantized=True)
    table = torch.arange(rows // 16, dtype=torch.int32, device=DEV).view(1, 1, -1)
    zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    x = x.to(DEV).view(1, 1, rows, 1, d)
    cache.write(x, x, table, zero)
    got = cache.k_pages.double() * cache.k_scales.double()[..., None]
    assert torch.equal(got.view(rows, d), quantise(x.view(rows, d)))


@pytest.mark.parametrize("quantized", [False, True])
def test_rows_that_are_not_finite(quantized):
    import wide_compiler as wc
    cache = wc.WidePagedCache(4, 8, 2, 32, dtype=torch.bfloat16, quantized=quantized)
    x = torch.randn(1, 1, 10, 2, 32, generator=gen(43)).to(DEV, torch.bfloat16)
    x[0, 0, 3, 0, 5], x[0, 0, 4, 1, 0], x[0, 0, 5, 0] = float("nan"), float("-inf"), 0
    table = torch.tensor([[[2, 0]]], dtype=torch.int32, device=DEV)
    zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    cache.write(x, x, table, zero)
    k, v = cache.read(table, zero + 10, 10)
    if not quantized:
        assert torch.equal(k.view(torch.int16), x.view(torch.int16)) and torch.equal(v.view(torch.int16), x.view(torch.int16))
        return
    bad = torch.isnan(quantise(x))
    assert torch.equal(torch.isnan(k), bad) and bad.any() and not bad.all()
    assert torch.equal(k[~bad], quantise(x).to(torch.bfloat16)[~bad]) and (k[0, 0, 5, 0] == 0).all()


@pytest.mark.parametrize("quantized", [False, True])
def test_strided_inputs_and_negative_starts(quantized):
    cache, k, v, table, start, count = _write(torch.bfloat16, quantized, 2, 2, 9, 4, 64, 16, 20, 47)
    start[1, 0] = -1
    cache.write(k, v, table, start, count)
    expect = cache.k_pages.clone(), cache.v_pages.clone()
    for way in (lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
                lambda t: torch.cat([t[..., :1], t], -1)[..., 1:], lambda t: t.transpose(3, 4).contiguous().transpose(3, 4)):
        cache.k_pages.zero_(), cache.v_pages.zero_()
        cache.write(way(k), way(v), table, start, count)
        assert torch.equal(cache.k_pages, expect[0]) and torch.equal(cache.v_pages, expect[1])
    cache.index_error()


@pytest.mark.parametrize("quantized", [False, True])
def test_tables_and_counts_out_of_range(quantized):
    """Nothing outside the pool is touched, the rest is written, the flag is raised once."""
    import wide_compiler as wc
    pages, page, h, d = 6, 8, 2, 32
    cache = wc.WidePagedCache(pages, page, h, d, dtype=torch.bfloat16, quantized=quantized)
    x = torch.randn(1, 1, 20, h, d, generator=gen(53)).to(DEV, torch.bfloat16)
    zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    for table, start, count, good in (([1, pages, 3], 0, None, [*range(8), *range(16, 20)]),
                                      ([1, -5, 3], 0, None, [*range(8), *range(16, 20)]),
                                      ([4, 2], 0, None, [*range(16)]),
                                      ([4, 2, 0], 0, 25, [*range(20)]),
                                      ([4, 2, 0], 2 ** 31 - 10, None, [])):
        t = torch.tensor([[table]], dtype=torch.int32, device=DEV)
        cache.k_pages.zero_(), cache.v_pages.zero_()
        cache.write(x, x, t, zero + start, None if count is None else zero + count)
        with pytest.raises(IndexError):
            cache.index_error()
        k, _ = cache.read(t, zero + min(20, len(table) * page), 20)
        ref = (quantise(x).to(x.dtype) if quantized else x).clone()
        keep = torch.zeros(20, dtype=torch.bool, device=DEV)
        keep[good] = True
        ref[:, :, ~keep] = 0
        assert torch.equal(k, ref)
        cache._err.zero_()
    k, _ = cache.read(torch.tensor([[[4, 2, 0]]], dtype=torch.int32, device=DEV), zero + 21, 20)
    with pytest.raises(IndexError):
        cache.index_error()


def test_empty_calls():
    import wide_compiler as wc
    cache = wc.WidePagedCache(2, 8, 2, 32)
    e = torch.zeros(1, 2, 0, 2, 32, device=DEV, dtype=torch.bfloat16)
    i = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    t = torch.zeros(1, 2, 0, dtype=torch.int32, device=DEV)
    cache.write(e, e, t, i)
    k, v = cache.read(t, i, 0)
    assert k.shape == (1, 2, 0, 2, 32)
    k, v = cache.read(t, i, 5)
    assert (k == 0).all() and k.shape == (1, 2, 5, 2, 32)
    cache.index_error()


def test_write_and_read_in_a_graph():
    cache, k, v, table, start, count = _write(torch.bfloat16, True, 2, 2, 6, 2, 64, 8, 20, 59)
    lens, most = start + count, int((start + count).max())
    cache.write(k, v, table, start, count)
    cache.read(table, lens, most)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, table, start, count)
        rk, rv = cache.read(table, lens, most)
    for step in range(3):
        k.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        a, c = rk.clone(), rv.clone()
        cache.write(k, v, table, start, count)
        ek, ev = cache.read(table, lens, most)
        assert torch.equal(a, ek) and torch.equal(c, ev)


@pytest.mark.parametrize("quantized", [False, True])
def test_a_table_without_entries(quantized):
    """Nothing to follow: what is asked of it is reported and reads as zeros, what isn't asked is fine."""
    import wide_compiler as wc
    cache = wc.WidePagedCache(4, 16, 2, 64, quantized=quantized)
    table = torch.zeros(2, 3, 0, dtype=torch.int32, device=DEV)
    k = torch.randn(2, 3, 5, 2, 64, device=DEV, dtype=torch.bfloat16)
    q = torch.randn(2, 3, 4, 64, device=DEV, dtype=torch.bfloat16)
    none, some = (torch.full((2, 3), x, dtype=torch.int32, device=DEV) for x in (0, 2))
    for lens in (none, some):
        for call in (lambda: cache.write(k, k, table, none, lens), lambda: cache.read(table, lens, 5),
                     lambda: (cache.attend(q, table, lens),)):
            out = call()
            assert out is None or all((o == 0).all() for o in out)
            if lens is some:
                with pytest.raises(IndexError):
                    cache.index_error()
            cache.index_error()
    assert (cache.k_pages == 0).all() and (cache.v_pages == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_codes_of_the_largest_values_are_finite(dtype):
    """A row that holds the type's largest value reads back as that value, to a unit of fp32's and its own last place, and
    the others as multiples of 1/127 of it, half of one off."""
    import wide_compiler as wc
    top = torch.finfo(dtype).max
    x = torch.linspace(-1, 1, 64).to(dtype).double() * top
    x[0], x[63], x[5] = -top, top, 0
    x = x.to(dtype).to(DEV).view(1, 1, 1, 1, 64)
    cache = wc.WidePagedCache(1, 16, 1, 64, dtype=dtype, quantized=True)
    table, start = torch.zeros(1, 1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    cache.write(x, x / 2, table, start)
    k, v = cache.read(table, start + 1, 1)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()
    for got, ref in ((k.double(), x.double()), (v.double(), x.double() / 2)):
        big = ref.abs().max()
        assert ((got - ref).abs() <= big * (1 / 254 + torch.finfo(dtype).eps + 2.0 ** -22)).all()
        assert ((got[..., [0, 63]] - ref[..., [0, 63]]).abs() <= big * (torch.finfo(dtype).eps + 2.0 ** -22)).all()


def test_sequences_that_take_no_part_raise_nothing():
    """A sequence of negative start is left out, whatever its count says; a count beyond the rows of another is reported."""
    cache, k, v, table, start, count = _write(torch.bfloat16, False, 2, 2, 5, 2, 64, 16, 9, 71)
    start[0, 1], count[0, 1] = -1, 99
    before = cache.k_pages.clone()
    expect = _expect(before, k, table, start, torch.where(start < 0, 0, count), 16, 64)
    cache.write(k, v, table, start, count)
    cache.index_error()
    assert torch.equal(cache.k_pages, expect)
    count[1, 1] = 6
    cache.write(k, v, table, start, count)
    with pytest.raises(IndexError):
        cache.index_error()
