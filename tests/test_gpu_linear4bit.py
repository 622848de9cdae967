"""WideLinear4bit (GPU) against 64 bits: types, rows around the tiles of 16 and 64, widths that end inside a tile or a
group, group sizes, zero points, bias, strided inputs, rows that aren't finite, graphs.

Tolerance: half a rounding step of the result, and what sums in fp32 lose: per term of a sum 2^-24 of what it adds up.
A group's sum holds codes (up to 15) and, in bf16, 128 more, times x; so the loss is bounded by 2^-24 times the number
of additions an output takes in one chain (columns / 4 waves / 8 in a product, and 16 more) times sum |x| (code + 128,
or + zero) scale."""

import pytest
import torch

from tests._serve import HALF, within
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _layer(n, k, o, group, zeros, bias, dtype, seed):
    import wide_compiler as wc
    g = gen(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, o, (k + 1) // 2), generator=g, dtype=torch.uint8)
    scales = (0.02 * (0.5 + torch.rand(n, o, groups, generator=g))).to(dtype)
    z = torch.randint(0, 16, (n, o, groups), generator=g, dtype=torch.uint8) if zeros else None
    b = torch.randn(n, o, generator=g).to(dtype) if bias else None
    mod = wc.WideLinear4bit.from_codes(codes.to(DEV), scales.to(DEV), in_features=k, group_size=group,
                                       zeros=None if z is None else z.to(DEV), bias=None if b is None else b.to(DEV))
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :k].double()
    at = torch.arange(k) // group
    zero = z.double()[..., at] if zeros else torch.full_like(c, 8.0)
    s = scales.double()[..., at]
    return mod, ((c - zero) * s).to(DEV), ((c + zero + (128 if dtype == torch.bfloat16 else 0)) * s).to(DEV), b


def _check(y, x, w, size, bias):
    n, k = x.shape[0], x.shape[-1]
    xd = x.double().reshape(n, -1, k)
    ref = torch.bmm(xd, w.transpose(1, 2).contiguous())
    # a row of size that isn't finite says nothing (its outputs aren't either)
    loss = torch.bmm(xd.abs(), size.transpose(1, 2).contiguous()).nan_to_num(0, 0, 0)
    if bias is not None:
        b = bias.to(DEV).double()[:, None]
        ref, loss = ref + b, loss + b.abs()
    within(y.reshape(ref.shape), ref, HALF[y.dtype], 2.0 ** -24 * (k / 32 + 20) * loss)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,m,k,o,zeros,bias", [
    (1, 1, 128, 16, False, False), (2, 1, 1000, 500, True, True), (3, 5, 256, 33, True, False), (1, 16, 64, 100, False, True),
    (2, 17, 520, 64, True, True), (1, 33, 37, 5, True, True), (1, 64, 1024, 130, False, False), (2, 65, 129, 48, True, False),
    (1, 200, 96, 17, True, True), (4, 1, 1, 1, True, True), (16, 3, 300, 500, True, True), (40, 16, 270, 600, True, False),
    (20, 20, 200, 300, True, True), (30, 30, 390, 600, True, True), (20, 50, 513, 320, True, True), (64, 64, 150, 1030, True, False)])
def test_linear4_sizes(n, m, k, o, zeros, bias, group, dtype):
    mod, w, size, b = _layer(n, k, o, group, zeros, bias, dtype, k + o + m)
    x = torch.randn(n, m, k, generator=gen(m)).to(DEV, dtype)
    y = mod(x)
    assert y.shape == (n, m, o) and y.dtype == dtype
    _check(y, x, w, size, b)
    assert torch.equal(mod.dequantize().double(), w.float().double()) or (mod.dequantize().double() - w).abs().max() <= 2.0 ** -23 * w.abs().max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,m", [(52, 3), (52, 20), (90, 5), (90, 32), (52, 90), (90, 70), (90, 64), (83, 5), (83, 32), (83, 60),
                                 (10, 20), (6, 50), (20, 3)])
@pytest.mark.parametrize("k", [150, 264, 600, 1160])
def test_linear4_many_layers(n, m, k, group, dtype):
    """Enough output rows for every form of the kernel, with widths of whole vectors and not."""
    mod, w, size, b = _layer(n, k, 600, group, True, True, dtype, n + m + k)
    x = torch.randn(n, m, k, generator=gen(m)).to(DEV, dtype)
    _check(mod(x), x, w, size, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_linear4_inputs_off_center(dtype):
    """All x of one sign (as behind a ReLU): the sums that are taken off again are at their largest."""
    mod, w, size, b = _layer(2, 4096, 64, 128, True, False, dtype, 3)
    x = (3 + torch.randn(2, 4, 4096, generator=gen(5))).to(DEV, dtype)
    _check(mod(x), x, w, size, b)


def test_linear4_batch_shapes_and_strides():
    mod, w, size, b = _layer(3, 256, 40, 64, True, True, torch.bfloat16, 7)
    x = torch.randn(3, 2, 5, 256, generator=gen(9)).to(DEV, torch.bfloat16)
    y = mod(x)
    assert y.shape == (3, 2, 5, 40)
    _check(y, x, w, size, b)
    packed = torch.randn(4, 3 * 256, generator=gen(11)).to(DEV, torch.bfloat16)       # channel-packed [B, N * I]
    view = packed.view(4, 3, 256).transpose(0, 1)
    assert torch.equal(mod(view), mod(view.contiguous()))
    wide = torch.zeros(3, 2, 5, 257, device=DEV, dtype=torch.bfloat16)
    wide[..., 1:] = x
    assert torch.equal(mod(wide[..., 1:]), y)
    assert torch.equal(mod(x.transpose(1, 2).contiguous().transpose(1, 2)), y)
    assert torch.equal(mod(x[..., None, :].expand(3, 2, 5, 2, 256))[..., 1, :], y)
    assert mod(x[:, :0]).shape == (3, 0, 5, 40)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_linear4_rows_not_finite(dtype):
    """What isn't finite stays in its own row of x."""
    mod, w, size, b = _layer(1, 300, 70, 32, True, False, dtype, 13)
    x = torch.randn(1, 20, 300, generator=gen(15)).to(DEV, dtype)
    expect = mod(x)
    x[0, 3, 5], x[0, 17, 299] = float("nan"), float("inf")
    y = mod(x)
    rest = [i for i in range(20) if i not in (3, 17)]
    assert torch.equal(y[:, rest], expect[:, rest])
    assert torch.isnan(y[0, 3]).all() and not torch.isfinite(y[0, 17]).any()


def test_linear4_from_modules_against_its_weights():
    import wide_compiler as wc
    lin = [torch.nn.Linear(200, 50).to(DEV, torch.bfloat16) for _ in range(3)]
    mod = wc.WideLinear4bit.from_modules(lin, group_size=32)
    w = mod.dequantize()
    orig = torch.stack([m.weight for m in lin]).float()
    # codes are at most half a step off, a step (max - min) / 15 and its rounding to bf16 (15 codes of 2^-8 / 2 steps)
    step = torch.nn.functional.pad(orig, (0, 24)).unflatten(-1, (7, 32))
    step = (step.amax(-1).clamp_min(0) - step.amin(-1).clamp_max(0)) / 15
    assert ((w - orig).abs().amax() <= (1.0 + 15 * 2.0 ** -8) * step.amax()).item()
    x = torch.randn(3, 2, 200, generator=gen(17)).to(DEV, torch.bfloat16)
    with torch.no_grad():
        y = mod(x)
    ref = torch.bmm(x.double(), w.double().transpose(1, 2).contiguous()) + mod.bias.double()[:, None]
    loss = torch.bmm(x.double().abs(), (w.double().abs() + 160 * mod.scales.amax().double()).transpose(1, 2).contiguous())
    within(y, ref, HALF[torch.bfloat16], 2.0 ** -24 * (200 / 32 + 20) * loss)


def test_linear4_state_dict_and_graph():
    import wide_compiler as wc
    mod, w, size, b = _layer(2, 384, 80, 128, True, True, torch.float16, 19)
    other = wc.WideLinear4bit(2, 384, 80, 128, bias=True, dtype=torch.float16).to(DEV)
    other.load_state_dict(mod.state_dict(), strict=True)
    x = torch.randn(2, 3, 384, generator=gen(21)).to(DEV, torch.float16)
    y = mod(x)
    assert torch.equal(other(x), y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mod(x)
    for _ in range(3):
        x.mul_(0.5)
        graph.replay()
        eager = mod(x)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@pytest.mark.parametrize("m", [1, 20, 70])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 3e-4), (torch.float16, 2e-6), (torch.bfloat16, 1e-36), (torch.float32, 1e-36)])
def test_linear4_small_weights(m, dtype, size):
    """Scales under the type's normal values (fp16) and next to them count as they are."""
    import wide_compiler as wc
    torch.manual_seed(7)
    lin = [torch.nn.Linear(200, 50, bias=False).to(DEV, dtype) for _ in range(2)]
    for layer in lin:
        torch.nn.init.uniform_(layer.weight, -size, size)
    mod = wc.WideLinear4bit.from_modules(lin, group_size=32)
    w = mod.dequantize().double()
    assert (w.abs().amax() >= size / 2).item()
    x = (8 * torch.randn(2, m, 200, generator=gen(17))).to(DEV, dtype)
    with torch.no_grad():
        y = mod(x)
    extra = 160 if dtype == torch.bfloat16 else 30          # codes, zero points and (bf16) 128, times the scale
    _check(y, x, w, w.abs() + extra * mod.scales.amax().double(), None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,m,k,o", [(1, 1, 512, 200), (3, 5, 4100, 40), (2, 20, 1000, 300), (90, 8, 600, 300), (52, 40, 390, 600), (20, 70, 300, 300)])
def test_linear4_weights_of_zero_take_no_part(n, m, k, o, group, dtype):
    """Where a column's codes are their zero points, nothing of x counts, however large it is, and what x sums up to
    counts nowhere: the loss is 2^-24 of the sum of |x w| for each addition, as above."""
    import wide_compiler as wc
    g = gen(k + m)
    groups, at = -(-k // group), torch.arange(k) // group
    codes = torch.randint(0, 16, (n, o, k), generator=g, dtype=torch.uint8)
    z = torch.randint(0, 16, (n, o, groups), generator=g, dtype=torch.uint8)
    none = torch.rand(k, generator=g) < 0.05
    none[7], none[k - 1], none[k - 2] = True, True, False
    codes = torch.where(none, z[..., at], codes)
    scales = (0.02 * (0.5 + torch.rand(n, o, groups, generator=g))).to(dtype)
    even = torch.nn.functional.pad(codes, (0, k % 2))
    mod = wc.WideLinear4bit.from_codes((even[..., 0::2] | even[..., 1::2] << 4).to(DEV), scales.to(DEV), in_features=k,
                                       group_size=group, zeros=z.to(DEV))
    w = ((codes.double() - z.double()[..., at]) * scales.double()[..., at]).to(DEV)
    assert (w[..., none.to(DEV)] == 0).all()
    x = 3 + torch.randn(n, m, k, generator=g)
    x[..., none] = 3e4 if dtype == torch.float16 else 1e37
    x = x.to(DEV, dtype)
    _check(mod(x), x, w, w.abs(), None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 20, 70])
def test_linear4_infinities_in_16_bits(m, dtype):
    """An infinity in x comes out as the formula has it: of its weights' sign, NaN where one is zero."""
    mod, w, size, b = _layer(2, 500, 300, 64, True, True, dtype, 23)
    x = torch.randn(2, m, 500, generator=gen(m)).to(DEV, dtype)
    x[0, 0, 77], x[1, m // 2, 499] = float("inf"), -float("inf")
    ref = torch.stack([(x[i].double()[:, None] * w[i]).sum(-1) for i in range(2)]) + b.to(DEV).double()[:, None]
    y = mod(x)
    assert torch.equal(torch.isnan(y), torch.isnan(ref)) and torch.equal(torch.isinf(y), torch.isinf(ref))
    assert torch.equal(y[torch.isinf(ref)].double(), ref[torch.isinf(ref)]) and 0 < torch.isinf(ref).sum() < 600


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,o,m,k", [
    (1, 600, 1, 2999), (1, 600, 1, 4097), (1, 600, 33, 4999), (1, 600, 5, 8192), (1, 600, 1, 8191),      # one tile of outputs
    (4, 2100, 1, 4999), (4, 4096, 3, 4096), (4, 4096, 1, 8191), (5, 2048, 9, 2047),                      # two, 8 and 4 waves
    (16, 2048, 1, 8192), (16, 2048, 3, 4999), (16, 2048, 7, 8191),                                       # chunks of 16 tiles
    (32, 2048, 16, 4097), (32, 2048, 50, 2056), (9, 2000, 70, 4097)])                                    # 16 and 8 waves
def test_linear4_long_columns(n, o, m, k, group, dtype):
    """Every form's loops over the columns come round again, with rows of x that are whole vectors and not; a chain of
    additions as above, each off by 2^-24 of the sum of |x w|."""
    import wide_compiler as wc
    g = torch.Generator(device=DEV).manual_seed(n + o + m + k)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, o, (k + 1) // 2), generator=g, dtype=torch.uint8, device=DEV)
    scales = (0.02 * (0.5 + torch.rand(n, o, groups, generator=g, device=DEV))).to(dtype)
    z = torch.randint(0, 16, (n, o, groups), generator=g, dtype=torch.uint8, device=DEV)
    mod = wc.WideLinear4bit.from_codes(codes, scales, in_features=k, group_size=group, zeros=z)
    x = torch.randn(n, m, k, generator=g, device=DEV).to(dtype)
    y = mod(x)
    at = torch.arange(k, device=DEV) // group
    for i in range(n):
        c = torch.stack((codes[i] & 15, codes[i] >> 4), -1).flatten(-2)[:, :k].double()
        w = ((c - z[i].double()[:, at]) * scales[i].double()[:, at])[None]
        _check(y[i:i + 1], x[i:i + 1], w, w.abs(), None)


def test_linear4_packs_one_model_at_a_time():
    """What packing takes beside the weights does not grow with the number of models: of 32, at most 4 bytes a weight with
    the packed half byte, where one model's own passes through fp32, its codes and their nibbles take 20 and more."""
    import wide_compiler as wc
    n, d = 32, 1024
    lin = [torch.nn.Linear(d, d, bias=False, device=DEV, dtype=torch.bfloat16) for _ in range(n)]
    codes = torch.randint(0, 256, (n, d, d // 2), dtype=torch.uint8, device=DEV)
    scales = torch.ones(n, d, d // 128, device=DEV)
    for make in (lambda: wc.WideLinear4bit.from_modules(lin), lambda: wc.WideLinear4bit.from_codes(codes, scales, in_features=d)):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        mod = make()
        torch.cuda.synchronize()
        assert torch.cuda.max_memory_allocated() - before <= 4 * n * d * d
        del mod
