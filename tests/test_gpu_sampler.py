"""Sampling (GPU) against the definition in 64 bits, row by row."""

import pytest
import torch

from tests._answer import draw
from tests._util import gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = float("inf")


def _logits(n, b, v, seed, dtype, spread=2.0):
    g = gen(seed)
    x = torch.randn(n, b, v, generator=g) * spread
    x[..., torch.randint(0, v, (5,), generator=g)] += 6
    return x.to(dtype)


def _check(sampler, x, u, rules, **given):
    with torch.no_grad():
        got = sampler(x.to(DEV), u.to(DEV), **{k: t.to(DEV) for k, t in given.items()}).cpu()
    assert got.shape == u.shape and got.dtype == torch.int64
    for at in torch.cartesian_prod(*(torch.arange(s) for s in u.shape)).view(-1, u.dim()).tolist():
        at = tuple(at)
        rule = {k: (r[at[0]] if isinstance(r, (list, tuple)) else r) for k, r in rules.items()}
        rule.update({k: t.expand(u.shape)[at].item() for k, t in given.items()})
        want = draw(x[at], u[at].item(), **rule)
        assert got[at].item() == want, (at, rule, got[at].item(), want)


RULES = [dict(), dict(temperature=0.0), dict(temperature=0.25), dict(top_k=1), dict(top_k=7), dict(top_p=0.9), dict(top_p=0.0),
         dict(min_p=0.05), dict(min_p=1.0), dict(temperature=1.7, top_k=50, top_p=0.8, min_p=0.01), dict(top_k=40, top_p=0.5),
         dict(temperature=5.0, top_p=0.99), dict(temperature=30.0, top_k=3000), dict(temperature=1e-3, top_p=0.7), dict(temperature=INF, top_k=9)]


# one logit, pieces of a vector, odd sizes, one and several pieces a thread, segments that end early
@pytest.mark.parametrize("v", [1, 2, 7, 64, 1000, 1025, 8191, 8192, 20011, 131072, 200003])
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens(v, dtype):
    import wide_compiler as wc
    n, b = 3, 2
    x = _logits(n, b, v, v, dtype)
    for i, rules in enumerate(RULES):
        u = torch.rand(n, b, generator=gen(i))
        _check(wc.WideSampler(n, **rules).to(DEV), x, u, rules)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rules", [dict(), dict(top_k=3), dict(top_k=5, top_p=0.5), dict(top_p=0.5), dict(min_p=1.0), dict(temperature=0.0)])
def test_equal_values_go_by_their_place(rules, dtype):
    import wide_compiler as wc
    for v in (1, 5, 64, 3000):
        for x in (torch.zeros(1, 4, v), torch.arange(v).flip(0).div(7, rounding_mode="floor").expand(1, 4, v).float() * 0.5,
                  torch.randint(0, 3, (1, 4, v), generator=gen(v)).float()):
            u = torch.tensor([[0.0, 0.3, 0.77, 1 - 2.0 ** -24]])
            _check(wc.WideSampler(1, **rules).to(DEV), x.to(dtype), u, rules)


def test_every_token_has_its_share():
    """u on a grid of 1 / 64: weights 1, 2, 4, ... of a sum of 63 each get as many of the 63 grid steps."""
    import wide_compiler as wc
    x = torch.log(torch.tensor([4.0, 1.0, 32.0, 2.0, 16.0, 8.0])).expand(1, 63, 6)
    u = ((torch.arange(63) + 0.5) / 63)[None]
    with torch.no_grad():
        got = wc.WideSampler(1).to(DEV)(x.to(DEV), u.to(DEV)).cpu()
    assert torch.bincount(got[0], minlength=6).tolist() == [4, 1, 32, 2, 16, 8]
    assert (got[0].diff() >= 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan(dtype):
    import wide_compiler as wc
    x = torch.randn(1, 9, 300, generator=gen(1))
    x[0, 0] = -INF
    x[0, 1] = float("nan")
    x[0, 2, :299] = -INF
    x[0, 3, ::2] = float("nan")
    x[0, 4, [5, 90, 250]] = INF
    x[0, 5, :] = -INF
    x[0, 5, [3, 8]] = torch.finfo(torch.float16).min
    x[0, 6, 1:] = torch.finfo(torch.float16).min
    x[0, 7, :150] = -INF
    x[0, 8, 7] = float("nan")
    for rules in RULES:
        _check(wc.WideSampler(1, **rules).to(DEV), x.to(dtype), torch.rand(1, 9, generator=gen(2)), rules)


def test_the_ends_of_u():
    import wide_compiler as wc
    x = _logits(1, 6, 5000, 3, torch.float32)
    x[0, :, 0] = -INF
    x[0, :, -1] = -INF
    u = torch.tensor([[0.0, 1 - 2.0 ** -24, 1.0, -3.0, 2.0, 1e-30]])
    for rules in RULES:
        _check(wc.WideSampler(1, **rules).to(DEV), x, u, rules)


def test_values_far_apart_and_tiny():
    """Values that differ in the last bit of fp32, of 1e30 and of 1e-40, at temperatures as extreme."""
    import wide_compiler as wc
    base = torch.rand(2, 3, 777, generator=gen(4))
    for x, t in ((base * 1e30, 1e29), (base * 1e-40, 1e-40), (1e30 + base * 1e24, 1e24), (base, 1e-30), (base, 1e30), (-base * 1e38, 3e38)):
        for rules in (dict(), dict(top_p=0.6), dict(top_k=5), dict(min_p=0.9), dict(top_k=200, top_p=0.7)):
            _check(wc.WideSampler(2, temperature=t, **rules).to(DEV), x, torch.rand(2, 3, generator=gen(5)), dict(temperature=t, **rules))


def test_rules_of_models_and_of_rows():
    import wide_compiler as wc
    n, b, v = 3, 4, 700
    x = _logits(n, b, v, 6, torch.float32)
    u = torch.rand(n, b, generator=gen(7))
    rules = dict(temperature=[0.5, 1.0, 0.0], top_k=[0, 20, 5], top_p=[0.9, 1.0, 0.3], min_p=[0.0, 0.1, 0.0])
    s = wc.WideSampler(n, **rules).to(DEV)
    _check(s, x, u, rules)
    _check(s.to(torch.bfloat16), x, u, rules)               # the rules stay as they are
    _check(s, x, u, rules, temperature=torch.rand(n, b, generator=gen(8)) + 0.2, top_k=torch.randint(0, 30, (b,), generator=gen(9), dtype=torch.int32))
    _check(s, x, u, rules, top_p=torch.rand(n, 1, generator=gen(10)), min_p=torch.tensor(0.02))
    s.set(temperature=1.5, top_k=[1, 2, 3])
    _check(s, x, u, {**rules, "temperature": 1.5, "top_k": [1, 2, 3]})


def test_strides_and_batches():
    import wide_compiler as wc
    base = torch.randn(3, 5, 2, 1001, generator=gen(11))
    s = wc.WideSampler(2, top_p=0.8).to(DEV)
    u = torch.rand(5, 2, 3, generator=gen(12)).permute(1, 0, 2)
    with torch.no_grad():
        for x in (base.permute(2, 1, 0, 3)[..., 1:], base.permute(2, 1, 0, 3)[..., ::2], base.permute(2, 1, 0, 3)[..., :900]):
            got = s(x.to(DEV), u.to(DEV))
            on = base.to(DEV).permute(2, 1, 0, 3)
            view = on[..., 1:] if x.shape[-1] == 1000 else on[..., ::2] if x.shape[-1] == 501 else on[..., :900]
            assert torch.equal(s(view, u.to(DEV)), got)
            for i, j, k in ((0, 0, 0), (1, 4, 2), (0, 3, 1)):
                assert got[i, j, k].item() == draw(x[i, j, k], u[i, j, k].item(), top_p=0.8)
        t = torch.rand(2, 3, 5, generator=gen(13)).permute(0, 2, 1) + 0.5          # a rule of its own strides
        got = s(base.permute(2, 1, 0, 3).to(DEV), u.to(DEV), temperature=t.to(DEV))
        for i, j, k in ((0, 0, 0), (1, 4, 2), (1, 2, 1)):
            assert got[i, j, k].item() == draw(base[k, j, i], u[i, j, k].item(), temperature=t[i, j, k].item(), top_p=0.8)
        assert s(torch.zeros(2, 0, 9, device=DEV), torch.zeros(2, 0, device=DEV)).shape == (2, 0)


def test_many_rows():
    import wide_compiler as wc
    x, u = _logits(4, 300, 515, 14, torch.bfloat16), torch.rand(4, 300, generator=gen(15))
    _check(wc.WideSampler(4, temperature=0.9, top_p=0.95).to(DEV), x, u, dict(temperature=0.9, top_p=0.95))


def test_a_graph_replays_with_new_numbers_and_rules():
    import wide_compiler as wc
    s = wc.WideSampler(2, temperature=1.0, top_p=0.9).to(DEV)
    x, u = _logits(2, 5, 9001, 16, torch.float16).to(DEV), torch.rand(2, 5, device=DEV)
    with torch.no_grad():
        s(x, u)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = s(x, u)
        for rep in range(4):
            x.copy_(_logits(2, 5, 9001, 20 + rep, torch.float16))
            u.copy_(torch.rand(2, 5, generator=gen(rep)))
            if rep == 2:
                s.set(top_k=4, min_p=0.1)
            graph.replay()
            torch.cuda.synchronize()
            want = got.clone()
            assert torch.equal(s(x, u), want)


def test_on_another_stream():
    import wide_compiler as wc
    s = wc.WideSampler(1, top_k=30).to(DEV)
    x, u = _logits(1, 3, 50001, 17, torch.float32).to(DEV), torch.rand(1, 3, device=DEV)
    with torch.no_grad():
        want = s(x, u)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = s(x, u)
        torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("v", [185, 829, 8192, 30000])
@pytest.mark.parametrize("top_k", [50, 464, 1024, 1100])
def test_fewer_allowed_than_top_k(top_k, v):
    """Rows in which all but a few logits are banned by -infinity, under and over top_k, with each other filter."""
    import wide_compiler as wc
    for left in (1, 3, 49, 128, 129, 463, 900, 1090):
        if left > v:
            continue
        x = _logits(1, 6, v, left, torch.bfloat16)
        kept = torch.randperm(v, generator=gen(left))[:left]
        banned = torch.ones(v, dtype=torch.bool)
        banned[kept] = False
        x[..., banned] = -INF
        for i, rest in enumerate((dict(), dict(top_p=0.9), dict(min_p=0.02), dict(top_p=0.7, min_p=0.05, temperature=1.5))):
            rules = dict(top_k=top_k, **rest)
            _check(wc.WideSampler(1, **rules).to(DEV), x, torch.rand(1, 6, generator=gen(i)), rules)


@pytest.mark.parametrize("v", [200, 8192, 9001, 70001])
@pytest.mark.parametrize("min_p", [1e-3, 1e-6, 2.0 ** -33, 1e-12, 1e-15, 2.0 ** -70, 1e-38, 1e-45])
def test_a_small_min_p_filters_what_it_says(v, min_p):
    """Values either side of min_p's border, a part of it and powers of two apart, the lower ones at the lowest places, which
    u = 0 gives if they are kept: with each other filter, and at temperatures that are taken over the digits of the values."""
    import wide_compiler as wc
    g = gen(v)
    border = -torch.log(torch.tensor(min_p, dtype=torch.float32).double()).item()
    for t in (1.0, 0.6, 40.0, 200.0):
        off = torch.cat([-torch.logspace(1.5, -4, 40), torch.logspace(-4, 1.5, 40)])     # from far below the border up to far above it
        x = -border * t + torch.randn(1, 8, v, generator=g).double() * 0.01 - 50 * t
        x[..., 3:83] = -border * t + off.double() * t
        x[..., v // 2:v // 2 + 3] = 0.0
        x = (x.clamp_max(0.0) + 3.0).float()
        u = torch.tensor([[0.0, 1e-30, 2.0 ** -39, 1e-9, 0.2, 0.5, 0.99, 1 - 2.0 ** -24]])
        for rest in (dict(), dict(top_k=60), dict(top_k=4, top_p=0.999999), dict(top_p=0.9999999)):
            rules = dict(temperature=t, min_p=min_p, **rest)
            _check(wc.WideSampler(1, **rules).to(DEV), x[:, :1], u[:, :1], rules)
            if min_p >= 2.0 ** -33:                          # weights of many units: the sums, too, are those in 64 bits
                _check(wc.WideSampler(1, **rules).to(DEV), x, u, rules)


def _crowded(kind, b, v, seed, dtype):
    """Rows of which one bin of weights next to the cut holds more values than a workgroup lists."""
    g = gen(seed)
    if kind == "wide":                                       # a large vocabulary's usual spread
        x = torch.randn(1, b, v, generator=g) * 2
        x[..., torch.randint(0, v, (20,), generator=g)] += 6
    elif kind == "flat":                                     # all in a bin or two, the largest among them
        x = 3 + torch.randn(1, b, v, generator=g) * 1e-3
    elif kind == "dense":                                    # a third of them next to each other within a part of the bin
        x = torch.randn(1, b, v, generator=g)
        x[..., ::3] = 0.5 + torch.randn(1, b, (v + 2) // 3, generator=g) * 1e-6
        x[..., 5] = 3.0
    elif kind == "zeros":                                    # small values of both signs about zero, zeros of both signs among them
        x = torch.randn(1, b, v, generator=g) * 1e-3
        x[..., ::7], x[..., 1::7] = 0.0, -0.0
        x[..., 11] = 2.0
    else:                                                    # far below: the last bin holds nearly all
        x = torch.randn(1, b, v, generator=g) - 60
        x[..., 9] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("kind,v", [("wide", 131072), ("wide", 262144), ("flat", 8000), ("flat", 20011), ("dense", 8192), ("dense", 70001), ("zeros", 8191),
                                    ("zeros", 40009), ("far", 8000), ("far", 30000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_more_values_in_a_bin_than_a_list_holds(kind, v, dtype):
    import wide_compiler as wc
    b = 5
    x = _crowded(kind, b, v, v, dtype)
    for i, rules in enumerate((dict(top_p=0.95), dict(top_p=0.5), dict(top_p=0.999), dict(top_p=1e-3), dict(temperature=1.5, top_p=0.9),
                               dict(temperature=4.0, top_p=0.3), dict(top_p=0.95, min_p=0.02), dict(top_p=0.99, min_p=1e-4, temperature=2.0),
                               dict(top_p=0.9, top_k=5000), dict(top_p=0.95, top_k=3000, min_p=1e-3), dict(top_p=0.97, min_p=0.9),
                               dict(temperature=0.01, top_p=0.95), dict(min_p=0.9), dict(min_p=0.01, temperature=4.0), dict(min_p=1e-5),
                               dict(min_p=1e-26), dict(min_p=1e-3, top_p=0.9999), dict(min_p=0.999, top_k=4000), dict(min_p=1e-4, top_k=20000))):
        u = torch.rand(1, b, generator=gen(i))
        u[0, 0], u[0, 1] = 0.0, 1 - 2.0 ** -24
        _check(wc.WideSampler(1, **rules).to(DEV), x, u, rules)


def test_more_equal_values_than_a_list_holds():
    import wide_compiler as wc
    x = torch.randint(0, 8, (1, 4, 100003), generator=gen(1)).float() * 0.3
    x[0, 2:] = torch.randint(0, 60, (2, 100003), generator=gen(2)).float() * 0.03
    u = torch.tensor([[0.0, 0.37, 0.81, 1 - 2.0 ** -24]])
    for dtype in DTYPES:
        for rules in (dict(top_p=0.5), dict(top_p=0.95), dict(top_p=0.7, min_p=0.3), dict(top_p=0.8, top_k=4000), dict(temperature=2.0, top_p=0.99)):
            _check(wc.WideSampler(1, **rules).to(DEV), x.to(dtype), u, rules)


def test_usual_rows_take_no_longer_than_their_neighbours():
    """Top-p over a large vocabulary takes about as long whether the cut's bin of weights holds a thousand values (temperature
    0.7) or several (1.0 and 1.5)."""
    import wide_compiler as wc
    x = _crowded("wide", 64, 200003, 3, torch.bfloat16).to(DEV)
    u = torch.rand(1, 64, generator=gen(4)).to(DEV)

    def time(t):
        s = wc.WideSampler(1, temperature=t, top_p=0.95).to(DEV)
        at = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        times = []
        with torch.no_grad():
            for _ in range(9):
                at[0].record()
                for _ in range(5):
                    s(x, u)
                at[1].record()
                torch.cuda.synchronize()
                times.append(at[0].elapsed_time(at[1]))
        return sorted(times)[4]
    base = time(0.7)
    assert time(1.0) < 4 * base and time(1.5) < 4 * base, (base, time(1.0), time(1.5))
