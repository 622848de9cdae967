"""WideHeadNormRotary (GPU) against 64 bits: types, head dims on both sides of the vector widths, partial and no
rotation, both pairings, broadcast and far positions, strided inputs, rows that aren't finite, graphs.

Tolerance: half a rounding step of the result, and for the fp32 arithmetic 16 2^-24 (norm, weight, two products, a
sum, sine and cosine, their angle's 2^-25 of a turn times 2 pi) of the larger of the pair's magnitudes, plus (d + 4)
2^-24 / 2 of the value for the sum of squares."""

import pytest
import torch

from tests._serve import HALF, within
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ref(x, w, pos, rot, base, eps, inter):
    """The definition in 64 bits; x [n, b, t, h, d], w [n, d], pos [n, b, t]; and the magnitude a pair has."""
    x, n = x.double(), x.shape[0]
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double().view(n, 1, 1, 1, -1)
    out, size = y.clone(), y.abs()
    p = torch.arange(rot // 2, device=x.device)
    a = (pos.double()[..., None] * base ** (-2.0 * p.double() / max(rot, 1)))[..., None, :]
    i, j = (2 * p, 2 * p + 1) if inter else (p, p + rot // 2)
    out[..., i] = y[..., i] * a.cos() - y[..., j] * a.sin()
    out[..., j] = y[..., j] * a.cos() + y[..., i] * a.sin()
    size[..., i] = size[..., j] = y[..., i].abs() + y[..., j].abs()
    return out, size


def _check(got, x, w, pos, rot, base, eps, inter):
    ref, size = _ref(x, w, pos, rot, base, eps, inter)
    d = x.shape[-1]
    within(got, ref, HALF[got.dtype], (16 + (d + 4) / 2) * 2.0 ** -24 * size + 1e-42)


def _module(n, d, rot, base, inter, dtype, seed, eps=1e-6):
    import wide_compiler as wc
    mod = wc.WideHeadNormRotary(n, d, rotary_dim=rot, base=base, interleaved=inter, eps=eps).to(DEV)
    g = gen(seed)
    with torch.no_grad():
        mod.q_weight.copy_(1 + 0.3 * torch.randn(n, d, generator=g))
        mod.k_weight.copy_(1 + 0.3 * torch.randn(n, d, generator=g))
    return mod.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("n,b,t,hq,hk,d,rot", [
    (1, 1, 1, 1, 1, 64, 64), (2, 3, 5, 8, 2, 128, 128), (3, 1, 7, 4, 4, 80, 40), (2, 2, 33, 12, 3, 96, 96),
    (1, 2, 9, 3, 1, 256, 128), (2, 1, 4, 2, 2, 2, 2), (1, 3, 11, 5, 1, 18, 6), (2, 2, 3, 1, 7, 250, 250),
    (1, 1, 700, 40, 8, 128, 0), (2, 1, 3, 100, 30, 64, 62)])
def test_head_norm_sizes(n, b, t, hq, hk, d, rot, inter, dtype):
    mod = _module(n, d, rot, 10000.0, inter, dtype, d + t)
    g = gen(hq)
    q = (3 * torch.randn(n, b, t, hq, d, generator=g)).to(DEV, dtype)
    k = (3 * torch.randn(n, b, t, hk, d, generator=g)).to(DEV, dtype)
    pos = torch.randint(0, 5000, (n, b, t), generator=g).to(DEV)
    with torch.no_grad():
        qo, ko = mod(q, k, pos)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == dtype
    _check(qo, q, mod.q_weight, pos, rot, 10000.0, 1e-6, inter)
    _check(ko, k, mod.k_weight, pos, rot, 10000.0, 1e-6, inter)


@pytest.mark.parametrize("pos_dtype,far", [(torch.int32, 2 ** 31 - 1), (torch.int64, 2 ** 40), (torch.int64, -123456789)])
def test_head_norm_far_positions(pos_dtype, far):
    """A far position turns by its true angle: in fp64 the product with a frequency below 1 is off by 2^-53 of it."""
    n, d = 2, 64
    mod = _module(n, d, d, 500.0, False, torch.float32, 1)
    q = torch.randn(n, 1, 6, 3, d, generator=gen(2)).to(DEV)
    pos = (far - (1 if far > 0 else -1) * torch.arange(6)).to(DEV, pos_dtype).expand(n, 1, 6)
    with torch.no_grad():
        qo, _ = mod(q, q, pos)
    ref, size = _ref(q, mod.q_weight, pos, d, 500.0, 1e-6, False)
    within(qo, ref, HALF[torch.float32], ((16 + (d + 4) / 2) * 2.0 ** -24 + 8 * abs(far) * 2.0 ** -53) * size)


def test_head_norm_positions_broadcast_and_strides():
    n, b, t, hq, hk, d = 2, 3, 5, 4, 2, 64
    mod = _module(n, d, d, 10000.0, False, torch.bfloat16, 3)
    qkv = torch.randn(n, b, t, (hq + 2 * hk) * d, generator=gen(4)).to(DEV, torch.bfloat16)
    q, k = qkv[..., :hq * d].unflatten(-1, (hq, d)), qkv[..., hq * d:(hq + hk) * d].unflatten(-1, (hk, d))
    pos = torch.arange(7, 7 + t, device=DEV)
    with torch.no_grad():
        qo, ko = mod(q, k, pos)
        _check(qo, q, mod.q_weight, pos.expand(n, b, t), d, 10000.0, 1e-6, False)
        for p in (pos.expand(n, b, t).contiguous(), pos.to(torch.int32), pos.expand(b, t)):
            a, c = mod(q.contiguous(), k.contiguous(), p)
            assert torch.equal(a, qo) and torch.equal(c, ko)
        # heads before tokens, an odd offset, a last stride that isn't 1
        a, _ = mod(q.transpose(2, 3).contiguous().transpose(2, 3), k, pos)
        assert torch.equal(a, qo)
        odd = torch.empty(n, b, t, hq, d + 1, device=DEV, dtype=q.dtype)
        odd[..., 1:] = q
        a, _ = mod(odd[..., 1:], k, pos)
        assert torch.equal(a, qo)
        a, _ = mod(q.transpose(3, 4).contiguous().transpose(3, 4), k, pos)
        assert torch.equal(a, qo)
        one = torch.full((n, b, 1), 11, device=DEV)
        a, _ = mod(q, k, one)
        _check(a, q, mod.q_weight, one.expand(n, b, t), d, 10000.0, 1e-6, False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_head_norm_rows_of_zeros_and_not_finite(dtype):
    """A row of zeros stays zero; what isn't finite stays in its own row."""
    n, b, t, h, d = 1, 1, 4, 9, 64
    mod = _module(n, d, d, 10000.0, False, dtype, 5)
    q = torch.randn(n, b, t, h, d, generator=gen(6)).to(DEV, dtype)
    q[0, 0, 1, 3] = 0
    q[0, 0, 2, 4, 7] = float("nan")
    q[0, 0, 3, 5, 60] = float("inf")
    pos = torch.arange(t, device=DEV)
    with torch.no_grad():
        qo, _ = mod(q, q, pos)
    assert (qo[0, 0, 1, 3] == 0).all()
    assert torch.isnan(qo[0, 0, 2, 4]).all() and torch.isnan(qo[0, 0, 3, 5, 60])
    ok = torch.ones(t, h, dtype=torch.bool)
    ok[2, 4] = ok[3, 5] = False
    assert torch.isfinite(qo[0, 0][ok]).all()


def test_head_norm_from_modules_and_rms_norm():
    """Without rotation: torch's nn.RMSNorm of each model, in its fp32."""
    import wide_compiler as wc
    qn, kn = ([torch.nn.RMSNorm(48, eps=1e-5) for _ in range(3)] for _ in range(2))
    for m in (*qn, *kn):
        torch.nn.init.normal_(m.weight, 1.0, 0.2)
    mod = wc.WideHeadNormRotary.from_modules(qn, kn, rotary_dim=0).to(DEV)
    q, k = torch.randn(3, 2, 5, 4, 48, device=DEV), torch.randn(3, 2, 5, 1, 48, device=DEV)
    with torch.no_grad():
        qo, ko = mod(q, k, torch.zeros(1, dtype=torch.int64, device=DEV))
        for i in range(3):
            _check(qo[i:i + 1], q[i:i + 1], qn[i].weight[None].to(DEV), torch.zeros(1, 2, 5, device=DEV), 0, 1.0, 1e-5, False)
            _check(ko[i:i + 1], k[i:i + 1], kn[i].weight[None].to(DEV), torch.zeros(1, 2, 5, device=DEV), 0, 1.0, 1e-5, False)
        assert torch.allclose(qo[1], qn[1].to(DEV)(q[1]), rtol=1e-5, atol=1e-6)


def test_head_norm_empty_and_graph():
    mod = _module(2, 64, 64, 10000.0, False, torch.bfloat16, 7)
    q = torch.randn(2, 3, 0, 4, 64, device=DEV, dtype=torch.bfloat16)
    with torch.no_grad():
        assert mod(q, q, torch.zeros(0, dtype=torch.int64, device=DEV))[0].shape == q.shape
        q = torch.randn(2, 3, 1, 4, 64, device=DEV, dtype=torch.bfloat16)
        k = torch.randn(2, 3, 1, 0, 64, device=DEV, dtype=torch.bfloat16)
        pos = torch.randint(0, 100, (2, 3, 1), device=DEV)
        assert mod(q, k, pos)[1].shape == k.shape
        k = torch.randn(2, 3, 1, 2, 64, device=DEV, dtype=torch.bfloat16)
        mod(q, k, pos)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            qo, ko = mod(q, k, pos)
        for _ in range(3):
            pos.add_(17)
            q.mul_(1.5)
            graph.replay()
            a, c = mod(q, k, pos)
            torch.cuda.synchronize()
            assert torch.equal(a, qo) and torch.equal(c, ko)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_head_norm_from_modules_of_default_eps(dtype):
    """nn.RMSNorm without an eps, on rows as small as its default; torch rounds the norm and the product with the weight
    apart, two half steps more."""
    import wide_compiler as wc
    norms = [torch.nn.RMSNorm(64).to(DEV, dtype) for _ in range(2)]
    for m in norms:
        torch.nn.init.normal_(m.weight, 1.0, 0.2)
    mod = wc.WideHeadNormRotary.from_modules(norms, norms, rotary_dim=0)
    pos = torch.zeros(1, dtype=torch.int64, device=DEV)
    for size in (1.0, 1e-2, 1e-3):
        q = (size * torch.randn(2, 2, 5, 4, 64, generator=gen(9))).to(DEV, dtype)
        with torch.no_grad():
            qo, _ = mod(q, q, pos)
            _check(qo, q, mod.q_weight, torch.zeros(2, 2, 5, device=DEV), 0, 1.0, 2.0 ** -23, False)
            for i in range(2):
                within(qo[i], norms[i](q[i]).double(), 4 * HALF[dtype] + 72 * 2.0 ** -24, 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 0), (64, 32), (80, 12), (18, 6)])
def test_head_norm_columns_that_are_not_turned_stand_alone(d, rot, inter, dtype):
    """What isn't finite in a column from rotary_dim on shows there alone: a row with an infinity is NaN in that column and
    zero in the others that aren't turned, a weight that is infinite makes its own column infinite."""
    mod = _module(1, d, rot, 10000.0, inter, dtype, 11)
    q = torch.randn(1, 1, d, 3, d, generator=gen(12)).to(DEV, dtype)
    pos = torch.arange(d, device=DEV)
    rest = [c for c in range(rot, d)]
    for c in rest:
        q[0, 0, c, 1, c] = float("inf")
    with torch.no_grad():
        qo, _ = mod(q, q, pos)
        ref, _ = _ref(q, mod.q_weight, pos.expand(1, 1, d), rot, 10000.0, 1e-6, inter)
        for c in rest:
            assert torch.isnan(qo[0, 0, c, 1, c])
            assert (qo[0, 0, c, 1, [x for x in rest if x != c]] == 0).all()
        assert torch.equal(torch.isnan(qo), torch.isnan(ref))
        mod.k_weight[0, d - 1] = float("inf")
        _, ko = mod(q[:, :, :, :1], q[:, :, :, :1], pos)
    assert torch.isinf(ko[..., d - 1]).all() and torch.isfinite(ko[..., :d - 1]).all()


@pytest.mark.parametrize("inter", [False, True])
def test_head_norm_turns_by_the_whole_angle(inter):
    """Rows whose norm is exact (a quarter of their columns 2, the others 0) come out as 2 cos and 2 sin of the angle.  Two
    roundings each, the function's and its correction's: an independent one has a variance of u^2 / 12 for the unit u of the
    last place, which over all angles is 0.716 2^-48 / 12 on average, and a function that is off by up to a unit has
    0.16 u^2 at most.  Root mean square of the pair: sqrt(2 0.716 (0.16 + 1 / 12)) 2^-24 = 0.59 2^-24; an angle rounded
    to fp32 adds 0.7 2^-24, 0.9 in all.  The bar is 0.65."""
    n, b, t, h, d = 1, 4, 512, 8, 128
    import wide_compiler as wc
    mod = wc.WideHeadNormRotary(n, d, base=500.0, eps=0.0, interleaved=inter).to(DEV)
    pairs = torch.rand(n, b, t, h, d // 2, generator=gen(13)).argsort(-1) < d // 4    # half of the pairs
    q = torch.zeros(n, b, t, h, d)
    if inter:
        q[..., 0::2] = 2.0 * pairs
    else:
        q[..., :d // 2] = 2.0 * pairs
    pos = torch.randint(0, 100000, (n, b, t), generator=gen(14))
    with torch.no_grad():
        qo, _ = mod(q.to(DEV), q[..., :0, :].to(DEV), pos.to(DEV))
    assert torch.equal(q.square().mean(-1), torch.ones(n, b, t, h))
    ref, _ = _ref(q, torch.ones(n, d), pos, d, 500.0, 0.0, inter)
    off = ((qo.cpu().double() - ref).square().sum(-1) / (2 * 2 * pairs.sum(-1))).mean().sqrt().item()
    assert off <= 0.65 * 2.0 ** -24, off / 2.0 ** -24
