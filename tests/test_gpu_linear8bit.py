"""Products in 8-bit integers (GPU) against the definition in 64 bits."""

import pytest
import torch

from tests._answer import linear8
from tests._serve import HALF, within
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _module(n, k, o, dtype, seed=0, bias=True):
    import wide_compiler as wc
    g = gen(seed)
    codes = torch.randint(-127, 128, (n, o, k), generator=g, dtype=torch.int8).to(DEV)
    scales = (torch.rand(n, o, generator=g) * 0.01 + 0.001).to(DEV)
    b = torch.randn(n, o, generator=g).to(DEV, dtype) if bias else None
    return wc.WideLinear8bit.from_codes(codes, scales, b), codes, scales, b


def _check(y, x, codes, scales, bias):
    """The sum is exact; its conversion, the scales' product, theirs with it and the bias are an fp32 rounding each.  What
    rounds past a type's largest value (fp16: 65504) is an infinity."""
    prod, ref = linear8(x, codes, scales, bias)
    ref = torch.where(torch.isinf(ref.to(x.dtype)), ref.to(x.dtype).double(), ref)
    within(y, ref, HALF[x.dtype] + 2 * 2.0 ** -24, 4 * 2.0 ** -24 * prod.abs().nan_to_num(0, 0, 0))


# rows either side of 16 (one tile), 64 and 128 (tiles of outputs), columns that end inside a tile, widths of one
@pytest.mark.parametrize("n,m,k,o", [
    (1, 1, 1, 1), (2, 5, 100, 37), (3, 16, 1000, 500), (4, 1, 2048, 96), (1, 17, 128, 16), (2, 33, 65, 1000), (2, 64, 300, 70),
    (3, 65, 130, 200), (1, 100, 640, 1030), (2, 200, 1000, 500), (1, 300, 2048, 520), (1, 3, 9000, 33), (1, 2, 131072, 16),
    (1, 1024, 256, 768), (2, 513, 384, 264), (40, 3, 72, 24)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_products(n, m, k, o, dtype):
    mod, codes, scales, bias = _module(n, k, o, dtype)
    x = (torch.randn(n, m, k, generator=gen(1)) * torch.logspace(-3, 3, m)[:, None]).to(DEV, dtype)
    with torch.no_grad():
        y = mod(x)
    assert y.shape == (n, m, o) and y.dtype == dtype
    _check(y, x, codes, scales, bias)


# several tiles of rows by workgroups of one tile of outputs, on both sides of 2048 of them; tiles of 64 x 128 on both sides
# of 256 of them; rows longer than 4096 and 8192 columns
@pytest.mark.parametrize("n,m,k,o", [(2, 31, 7008, 96), (1, 48, 8200, 304), (1, 129, 4100, 416), (1, 33, 200, 10930), (1, 33, 200, 10900),
                                     (2, 293, 700, 1004), (1, 500, 650, 4090), (1, 520, 650, 4090)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_few_tiles(n, m, k, o, dtype):
    mod, codes, scales, bias = _module(n, k, o, dtype)
    x = torch.randn(n, m, k, generator=gen(4)).to(DEV, dtype)
    with torch.no_grad():
        _check(mod(x), x, codes, scales, bias)


# codes of as many rows as there are compute units of 16, of lengths that registers hold and longer ones
@pytest.mark.parametrize("k", [200, 1100, 2100, 4200, 8300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_rows_of_any_length(k, dtype):
    mod, codes, scales, bias = _module(2, k, 40, dtype)
    x = torch.randn(2, 2100, k, generator=gen(5)).to(DEV, dtype)
    x[1, 2050, k - 1] = 1000.0                               # a row's largest in its last column
    with torch.no_grad():
        _check(mod(x), x, codes, scales, bias)
        # the same rows, their codes found by several workgroups
        assert torch.equal(mod(x[:, 2040:2060]), mod(x)[:, 2040:2060])


def test_large_tiles_at_the_edges():
    """Rows and outputs next to the largest tile's, both ends of it ragged."""
    for m, k, o in ((2049, 512, 1025), (2304, 384, 2303)):
        mod, codes, scales, bias = _module(1, k, o, torch.bfloat16)
        x = torch.randn(1, m, k, generator=gen(2)).to(DEV, torch.bfloat16)
        with torch.no_grad():
            _check(mod(x), x, codes, scales, bias)


# as many of the largest tiles as there are compute units, fewer and more, both ends ragged; a stage or two of columns, and many
@pytest.mark.parametrize("n,m,k,o", [(8, 1040, 65, 1030), (8, 1040, 700, 1030), (8, 2049, 128, 1025), (8, 2049, 390, 1025), (1, 3000, 1000, 3300)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rounds_of_large_tiles(n, m, k, o, dtype):
    mod, codes, scales, bias = _module(n, k, o, dtype)
    x = torch.randn(n, m, k, generator=gen(6)).to(DEV, dtype)
    with torch.no_grad():
        _check(mod(x), x, codes, scales, bias)


def test_the_largest_sums():
    """All codes 127, as many columns as are allowed: 2 114 060 288 < 2^31, whatever order it is summed in."""
    import wide_compiler as wc
    codes = torch.full((1, 17, 131072), 127, dtype=torch.int8, device=DEV)
    codes[0, 1] = -127
    mod = wc.WideLinear8bit.from_codes(codes, torch.ones(1, 17, device=DEV))
    for m in (1, 20, 200):
        x = torch.full((1, m, 131072), 3.0, device=DEV)
        with torch.no_grad():
            _check(mod(x), x, codes, torch.ones(1, 17, device=DEV), None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_do_not_know_each_other(dtype):
    """Whatever batch a row is in, its result has the same bits."""
    mod, *_ = _module(2, 520, 264, dtype)
    x = torch.randn(2, 700, 520, generator=gen(3)).to(DEV, dtype)
    with torch.no_grad():
        y = mod(x)
        for m in (1, 9, 30, 100):
            at = torch.randperm(700, generator=gen(m))[:m].to(DEV)
            assert torch.equal(mod(x[:, at].contiguous()), y[:, at])


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    mod, codes, scales, bias = _module(2, 96, 40, dtype)
    base = torch.randn(5, 7, 2, 3 * 96 + 1, generator=gen(4)).to(DEV, dtype)
    with torch.no_grad():
        for x in (base.permute(2, 0, 1, 3)[..., 96:192], base.permute(2, 1, 0, 3)[..., 1:97], base.permute(2, 0, 1, 3)[:, 1, :, :96],
                  base.permute(2, 0, 1, 3)[..., 0:192:2], base[:1, :1].permute(2, 0, 1, 3)[..., 5:101]):
            y = mod(x)
            assert y.shape == (*x.shape[:-1], 40)
            _check(y, x.contiguous(), codes, scales, bias)
        wide = base.permute(2, 0, 1, 3)[:, :1, :1, :96].expand(2, 4, 5, 96)
        _check(mod(wide), wide.contiguous(), codes, scales, bias)


def test_values_next_to_a_half_go_to_even():
    """Rows whose largest is 127 have scale 1: k + 1/2 to the even neighbour, and what lies an fp32 step beside it."""
    halves = torch.arange(-126, 126).float() + 0.5
    row = torch.cat([torch.tensor([127.0]), halves, torch.nextafter(halves, torch.tensor(200.0)), torch.nextafter(halves, torch.tensor(-200.0))])
    import wide_compiler as wc
    k = len(row)
    mod = wc.WideLinear8bit.from_codes(torch.eye(k, dtype=torch.int8, device=DEV)[None], torch.ones(1, k, device=DEV))
    scale = 2.0 ** torch.arange(-100, 101, 50)
    x = (row * scale[:, None])[None].to(DEV)
    with torch.no_grad():
        y = mod(x)[0].double() / scale.double().to(DEV)[:, None]
    assert torch.equal(y, torch.round(row.double()).to(DEV).expand_as(y))


@pytest.mark.parametrize("m", [3, 40, 300])
def test_special_rows(m):
    mod, codes, scales, bias = _module(2, 200, 50, torch.float32)
    x = torch.randn(2, m, 200, generator=gen(5)).to(DEV)
    x[0, 0] = 0
    x[0, 1, 7] = float("inf")
    x[0, 2, 199] = float("nan")
    x[1, 0] *= 1e-44                                        # under the smallest scale: codes of 0
    x[1, 1] = 3.4028234663852886e38
    x[1, 2, :] = 0
    x[1, 2, 3] = -1e-39
    with torch.no_grad():
        y = mod(x)
    assert torch.isnan(y[0, 1:3]).all() and torch.equal(y[0, 0], bias[0])
    ok = torch.ones(2, m, dtype=torch.bool, device=DEV)
    ok[0, 1:3] = False
    ok[1, 1] = False
    prod, ref = linear8(x, codes, scales, bias)
    assert not ((y.double() - ref)[ok].abs() > (4 * 2.0 ** -24 * prod.abs() + 3 * 2.0 ** -24 * ref.abs())[ok]).any()
    # the largest value's scale is a step less than a 127th of it (2^-23 of the products), its codes 127; sums of them pass
    # fp32's range as the formula's do
    far = ref[1, 1].abs() > 3.3e38
    assert ((y[1, 1].double() - ref[1, 1]).abs() <= 2.0 ** -21 * ref[1, 1].abs())[~far].all() and (y[1, 1][far].sign() == ref[1, 1][far].sign()).all()


def test_nothing_to_do():
    mod, *_ = _module(2, 16, 8, torch.float32)
    with torch.no_grad():
        assert mod(torch.zeros(2, 0, 16, device=DEV)).shape == (2, 0, 8)
        assert mod(torch.zeros(2, 3, 0, 16, device=DEV)).shape == (2, 3, 0, 8)


def test_from_modules():
    """Weights come back within half a step of a 127th of their row's largest."""
    import wide_compiler as wc
    torch.manual_seed(1)
    mods = [torch.nn.Linear(200, 56).to(DEV, torch.bfloat16) for _ in range(3)]
    wide = wc.WideLinear8bit.from_modules(mods)
    w = torch.stack([m.weight for m in mods]).double()
    assert not ((wide.dequantize().double() - w).abs() > w.abs().amax(-1, keepdim=True) / 254 * (1 + 2.0 ** -20)).any()
    x = torch.randn(3, 6, 200, generator=gen(6)).to(DEV, torch.bfloat16)
    with torch.no_grad():
        prod, ref = linear8(x, torch.round(wide.dequantize().double() / wide.scales.double()[..., None]), wide.scales, wide.bias)
        within(wide(x), ref, HALF[torch.bfloat16] + 2.0 ** -23, 4 * 2.0 ** -24 * prod.abs())


def test_another_stream_a_graph_and_two_calls_at_once():
    mod, codes, scales, bias = _module(2, 256, 128, torch.bfloat16)
    xs = [torch.randn(2, m, 256, generator=gen(m)).to(DEV, torch.bfloat16) for m in (1, 48, 400)]
    with torch.no_grad():
        want = [mod(x) for x in xs]
        side = [torch.cuda.Stream() for _ in xs]
        for s in side:
            s.wait_stream(torch.cuda.current_stream())
        got = []
        for s, x in zip(side, xs):
            with torch.cuda.stream(s):
                got.append(mod(x))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        graphs = []
        for x in xs:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                y = mod(x)
            graphs.append((graph, y))
        for rep in range(3):
            for x in xs:
                x.copy_(torch.randn(x.shape, generator=gen(100 + rep)))
            for graph, _ in graphs:
                graph.replay()
            for x, (_, y) in zip(xs, graphs):
                assert torch.equal(mod(x), y)
            torch.cuda.synchronize()


def test_gradients_are_refused():
    mod, *_ = _module(1, 16, 8, torch.float32)
    with pytest.raises(RuntimeError):
        mod(torch.zeros(1, 2, 16, device=DEV, requires_grad=True))


# a row, few rows, tiles of 64 x 128 in six stages and in three, of 128 x 128, the largest
@pytest.mark.parametrize("n,m,k,o", [(2, 3, 200, 52), (2, 40, 200, 50), (1, 300, 130, 2100), (8, 60, 70, 4099), (8, 200, 70, 2100), (8, 1040, 65, 1030)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_and_scales_of_any_size(n, m, k, o, dtype):
    """Rows of 1e-38 to 1e38 against scales of 1e-40 to 1e38: the scales' product may be far under or over fp32's range where
    the result is not.  The same roundings as elsewhere: the sum's, the scales' product's, theirs with it and the result's."""
    import wide_compiler as wc
    g = gen(7)
    codes = torch.randint(-127, 128, (n, o, k), generator=g, dtype=torch.int8).to(DEV)
    scales = torch.logspace(-40, 38, o, dtype=torch.float64).float().expand(n, o)[:, torch.randperm(o, generator=g)].contiguous().to(DEV)
    scales[:, 0], scales[:, 1] = 0.0, -3e-6
    x = torch.randn(n, m, k, generator=g).clamp(-3, 3).double() * torch.logspace(-38, 38, m, dtype=torch.float64)[torch.randperm(m, generator=g)][:, None]
    x[:, 1] = 0
    x = x.clamp(-3e38, 3e38).to(DEV, dtype)
    mod = wc.WideLinear8bit.from_codes(codes, scales)
    with torch.no_grad():
        y = mod(x)
    _check(y, x, codes, scales, None)
    assert (y[:, 1] == 0).all() and (y[..., 0] == 0).all()


def test_small_rows_of_usual_weights():
    """Rows of 1e-36 and 1e-37 of weights of 3e-4: outputs are normal numbers, right to the roundings of 1."""
    import wide_compiler as wc
    _, codes, scales, _ = _module(2, 256, 64, torch.float32, bias=False)
    scales = scales * 1e-3
    mod = wc.WideLinear8bit.from_codes(codes, scales)
    for m in (2, 20, 600):
        base = torch.randn(2, m, 256, generator=gen(m)).to(DEV)
        for size in (1.0, 1e-34, 1e-35, 1e-36, 1e-37):
            x = base * size
            with torch.no_grad():
                _check(mod(x), x, codes, scales, None)


# (models, rows, columns, outputs) by the kernel that makes them (test_answer_api.py checks that it does): ragged rows and outputs,
# columns of one stage, of two and of several times the ring
FORMS = {
    "fused": [(3, 16, 960, 100), (2, 1, 1024, 17), (1, 3, 5000, 33)],
    "few": [(2, 16, 1100, 200), (1, 129, 700, 416), (3, 17, 65, 33)],
    "ring6": [(1, 300, 130, 2100), (2, 293, 900, 1004), (1, 40, 2000, 16400)],
    "ring3": [(8, 64, 2048, 4104), (9, 33, 200, 3800), (16, 49, 65, 2100), (11, 17, 130, 3000), (10, 60, 450, 3334)],
    "large": [(4, 2049, 512, 1025), (2, 2304, 384, 2303), (10, 257, 65, 2049)],
    "tiles": [(1, 2049, 512, 1025), (8, 200, 70, 2100), (3, 500, 300, 2100)],
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_kernel(form, dtype):
    for n, m, k, o in FORMS[form]:
        mod, codes, scales, bias = _module(n, k, o, dtype, seed=o)
        x = torch.randn(n, m, k, generator=gen(8)).to(DEV, dtype)
        x[:, m - 1, k - 1] = 9.0                             # the last row's largest in its last column
        with torch.no_grad():
            y = mod(x)
        _check(y, x, codes, scales, bias)
        # the same bits from a few of the rows
        at = torch.tensor([0, m // 2, m - 1], device=DEV)
        with torch.no_grad():
            assert torch.equal(mod(x[:, at].contiguous()), y[:, at])
