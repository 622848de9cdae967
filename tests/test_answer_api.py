"""The operators that draw many answers to the same prompts, without a GPU: their header and binding agree, the library
refuses bad arguments before any launch, the modules refuse tensors they do not take, 8-bit weights pack exactly."""

import ctypes
import hashlib
import os
import re
import shutil
import subprocess
import sys

import pytest
import torch

from tests.conftest import PKG, ROOT
from tests._util import gen

HEADER = os.path.join(ROOT, "include", "wc_answer_abi.h")
SAN_LIB = os.path.join(PKG, "wide_compiler", "libwide_hip_san.so")


@pytest.fixture(scope="module")
def answer():
    from wide_compiler import _answer
    _answer.lib()
    return _answer


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_binding_declares_what_the_header_does(answer):
    from wide_compiler import _serve
    declared = sorted(set(re.findall(r"\b(wc_[a-z0-9_]+)\s*\(", _text())))
    assert sorted(answer.SIGNATURES) == declared
    assert answer.lib().wc_answer_abi_version() == answer.ABI_VERSION
    for cls, name in ((answer._SharedAttnArgs, "wc_shared_attn_args"), (answer._Linear8Args, "wc_linear8_args"),
                      (answer._SampleArgs, "wc_sample_args")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _text(), flags=re.S).group(1)
        fields = []
        for decl in body.split(";"):
            words = decl.replace("const", " ").replace("*", " ").split()
            if not words:
                continue
            if words[0] == "wc_paged_cache":
                fields += [f for f, _ in _serve._PagedCache._fields_]
            else:
                fields += " ".join(words[1:]).replace(" ", "").split(",")
        assert [f for f, _ in cls._fields_] == fields, name


# a digest of include/wc_answer_abi.h without comments, per version
DECLARATIONS = {1: "28725dc905012c0f9bfb81c1d30350b6fedddc6be265c7f88cb398c4ef47813b"}


def test_every_change_of_the_header_has_a_version_of_its_own(answer):
    assert DECLARATIONS.get(answer.ABI_VERSION) == hashlib.sha256(" ".join(_text().split()).encode()).hexdigest()


def _fill(a, base, kw):
    for f, v in {**base, **kw}.items():
        setattr(a, f, v)
    return a


def test_library_refuses_bad_arguments(answer):
    lib, big = answer.lib(), (1 << 63) - 1
    error = lambda: lib.wc_last_error().decode()  # noqa: E731
    for name, (_, args) in answer.SIGNATURES.items():
        if len(args) == 2:
            assert getattr(lib, name)(None, None) == -1, name
        elif args:
            assert getattr(lib, name)(None) == -1, name

    def attend(**kw):
        a = _fill(answer._SharedAttnArgs(), dict(
            dtype=1, bits=0, n=1, b=4, pages=4, page_size=16, heads=2, head_dim=64, row=64, k_pages=4096, v_pages=4096,
            table=4096, table_len=3, table_stride=3, share=2, prefix_table=4096, prefix_len=5, prefix_stride=5,
            prefix_lengths=4096, q_heads=8, max_prefix=4000, max_length=400, q=4096, o=4096, lengths=4096, scale=0.1), kw)
        need = int(lib.wc_shared_attention_workspace_bytes(ctypes.byref(a)))
        if "workspace" not in kw and need > 0:
            a.workspace, a.workspace_bytes = 4096, need - 1
        return lib.wc_shared_attention(ctypes.byref(a), None), need
    assert attend()[0] == -6 and "workspace" in error()
    for kw in (dict(q_heads=3), dict(q_heads=-2), dict(share=0), dict(share=3), dict(share=-1), dict(max_prefix=-1), dict(max_length=-1),
               dict(prefix_len=-1), dict(head_dim=0), dict(n=-1)):
        assert attend(**kw) == (-2, -1), kw
    for kw in (dict(max_prefix=big), dict(max_length=big), dict(prefix_len=big), dict(q_heads=1 << 20), dict(row=512, dtype=0),
               dict(b=big - 1, share=1), dict(head_dim=300, row=304), dict(n=1 << 21, q_heads=8),
               dict(n=1 << 10, b=1 << 9, share=1, prefix_len=1 << 30, max_prefix=1 << 30)):
        assert attend(**kw) == (-5, -1), kw
    assert attend(dtype=7) == (-3, -1) and attend(bits=4) == (-3, -1) and attend(row=60)[0] == -2 and attend(row=68)[0] == -4
    assert attend(prefix_stride=-1) == (-6, -1)
    for kw, rc in ((dict(q=None), -1), (dict(prefix_lengths=None), -1), (dict(prefix_table=None), -1), (dict(lengths=None), -1),
                   (dict(o=4097), -4), (dict(prefix_table=4098), -4), (dict(k_pages=4104), -4), (dict(bits=8), -1),
                   (dict(workspace=4100, workspace_bytes=1 << 40), -4), (dict(workspace=None, workspace_bytes=1 << 40), -6)):
        assert attend(**kw)[0] == rc, kw
    assert attend(b=0) == (0, 0) and attend(q_heads=0) == (0, 0) and attend(n=0) == (0, 0)

    def linear(**kw):
        a = _fill(answer._Linear8Args(), dict(dtype=1, n=2, m=3, o=40, k=100, x=4096, x_rows_inner=3, codes=4096, scales=4096,
                                              y=4096), kw)
        need = int(lib.wc_linear8_workspace_bytes(ctypes.byref(a)))
        if "workspace" not in kw and need > 0:
            a.workspace, a.workspace_bytes = 4096, need - 1
        return lib.wc_linear8(ctypes.byref(a), None), need
    assert linear()[0] == -6 and "workspace" in error()
    assert linear(dtype=3) == (-3, -1) and linear(k=-1) == (-2, -1) and linear(k=0)[0] == -2 and linear(k=131073) == (-5, -1)
    assert linear(o=big) == (-5, -1) and linear(m=1 << 30) == (-5, -1) and linear(n=1 << 30) == (-5, -1)
    assert linear(m=1 << 20, o=1 << 20) == (-5, -1)
    assert linear(x_rows_inner=1 << 32)[0] == -5 and linear(x_rows_inner=0)[0] == -6
    assert linear(codes=4100)[0] == -4 and linear(scales=4098)[0] == -4 and linear(x=4097)[0] == -4 and linear(bias=4097)[0] == -4
    assert linear(workspace=4100, workspace_bytes=1 << 30)[0] == -4 and linear(workspace=None)[0] == -6
    assert linear(y=None)[0] == -1 and linear(m=0) == (0, 0) and linear(o=0) == (0, 0)

    def sample(**kw):
        a = _fill(answer._SampleArgs(), dict(dtype=1, n=2, m=3, v=100, logits=4096, x_rows_inner=3, u=4096, temperature=4096,
                                             top_k=4096, top_p=4096, min_p=4096, tokens=4096), kw)
        return lib.wc_sample(ctypes.byref(a), None), int(lib.wc_sample_workspace_bytes(ctypes.byref(a)))
    assert sample(dtype=3) == (-3, -1) and sample(m=-1) == (-2, -1) and sample(v=0)[0] == -2 and sample(v=1 << 30) == (-5, -1)
    assert sample(n=1 << 22) == (-5, -1) and sample(m=big) == (-5, -1) and sample(x_rows_inner=0)[0] == -6
    assert sample(x_rows_inner=1 << 32)[0] == -5
    for name in ("logits", "u", "temperature", "top_k", "top_p", "min_p", "tokens"):
        assert sample(**{name: None})[0] == -1 and sample(**{name: 4097})[0] == -4, name
    assert sample(tokens=4100)[0] == -4 and sample(n=0)[0] == 0 and sample(m=0)[0] == 0


def test_cpu_tensors_are_refused():
    import wide_compiler as wc
    for call in (lambda: wc.WideLinear8bit(1, 64, 16)(torch.zeros(1, 2, 64)),
                 lambda: wc.WideSampler(1)(torch.zeros(1, 2, 64), torch.zeros(1, 2))):
        with pytest.raises(RuntimeError, match="ROCm device tensors only"):
            call()


@pytest.fixture
def anywhere(monkeypatch):
    """Lets CPU tensors through the modules' checks, up to the launch, which must not be reached."""
    from wide_compiler import _answer, _hip

    def reached(*args, **kw):
        raise AssertionError("launched")
    monkeypatch.setattr(_hip, "require_device", lambda *a: None)
    for name in ("shared_attention", "linear8", "sample"):
        monkeypatch.setattr(_answer, name, reached)
        monkeypatch.setattr(_answer, name + "_workspace", lambda *a: 0)


def test_attend_shared_refusals(anywhere):
    import wide_compiler as wc
    pages = torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)
    cache = wc.WidePagedCache.from_pages(pages, pages)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    q, good = torch.zeros(2, 6, 4, 64, dtype=torch.bfloat16), (i(2, 3, 4), i(2, 3), i(2, 6, 2), i(2, 6))
    with torch.no_grad():
        with pytest.raises(AssertionError, match="launched"):
            cache.attend_shared(q, *good)
        for at, bad in ((0, i(2, 4, 4)), (0, i(1, 3, 4)), (0, i(2, 3, 4).long()), (0, i(2, 3)), (1, i(2, 2)), (1, i(2, 3).float()),
                        (1, i(2, 3, 1)), (2, i(2, 5, 2)), (2, i(2, 6, 2).long()), (3, i(2, 3)), (3, i(2, 6).long()), (0, i(2, 0, 4))):
            args = list(good)
            args[at] = bad
            with pytest.raises(RuntimeError):
                cache.attend_shared(q, *args)
        for bad in (q[..., :32], q[:, :, :3], q.half(), q[None], q[:, :4]):
            with pytest.raises(RuntimeError):
                cache.attend_shared(bad, *good)
        for kw in (dict(max_prefix=-1), dict(max_length=-1)):
            with pytest.raises(RuntimeError, match="negative"):
                cache.attend_shared(q, *good, **kw)
    with pytest.raises(RuntimeError, match="forward-only"):
        cache.attend_shared(q.requires_grad_(), *good)


def test_linear8_refusals(anywhere):
    import wide_compiler as wc
    for k in (0, 131073):
        with pytest.raises(ValueError):
            wc.WideLinear8bit(1, k, 16)
    with pytest.raises(TypeError):
        wc.WideLinear8bit(1, 64, 16, dtype=torch.float64)
    codes, scales = torch.zeros(2, 16, 64, dtype=torch.int8), torch.ones(2, 16)
    f = wc.WideLinear8bit.from_codes
    for kw in (dict(codes=codes.int()), dict(codes=codes[0]), dict(scales=scales[:, :8]), dict(scales=scales.half()),
               dict(bias=torch.zeros(2, 15)), dict(codes=codes - 128)):
        kw = dict(codes=codes, scales=scales) | kw
        with pytest.raises(ValueError):
            f(**kw)
    lin = lambda *a, **kw: torch.nn.Linear(*a, **kw)  # noqa: E731
    for mods in ([lin(4, 5), lin(5, 5)], [lin(4, 5), lin(4, 5, bias=False)], [lin(4, 5), lin(4, 5).half()]):
        with pytest.raises(ValueError):
            wc.WideLinear8bit.from_modules(mods)
    mod = f(codes, scales, torch.zeros(2, 16))
    x = torch.zeros(2, 3, 64)
    with pytest.raises(AssertionError, match="launched"):
        mod(x)
    for bad in (torch.zeros(2, 3, 32), torch.zeros(1, 3, 64), x.half(), torch.zeros(64)):
        with pytest.raises(RuntimeError):
            mod(bad)
    for name, t in (("packed", mod.packed[:, :, :, :32]), ("packed", mod.packed.int()), ("scale_bits", mod.scale_bits[:, :8]),
                    ("scale_bits", mod.scales), ("bias", torch.zeros(2, 15)), ("bias", torch.zeros(2, 16).half())):
        old = getattr(mod, name)
        setattr(mod, name, t)
        with pytest.raises(RuntimeError, match=name):
            mod(x)
        setattr(mod, name, old)
    with pytest.raises(RuntimeError, match="forward-only"):
        mod(x.requires_grad_())


@pytest.mark.parametrize("n,o,k", [(2, 500, 1000), (1, 16, 128), (3, 5, 37), (1, 33, 129), (2, 1, 1)])
def test_linear8_codes_pack_and_unpack_exactly(n, o, k):
    import wide_compiler as wc
    codes = torch.randint(-127, 128, (n, o, k), generator=gen(k), dtype=torch.int8)
    scales = torch.rand(n, o, generator=gen(o))
    mod = wc.WideLinear8bit.from_codes(codes, scales)
    want = codes.float() * scales[..., None]
    assert torch.equal(mod.dequantize(), want) and torch.equal(mod.half().dequantize(), want)
    # byte e of lane l of a tile: row l % 16, column 16 (l / 16) + e
    t, c, lane, e = 0, min(1, (k - 1) // 64), 21, 3
    row, col = t * 16 + lane % 16, c * 64 + 16 * (lane // 16) + e
    assert mod.packed[0, t, c, lane, e] == (codes[0, row, col] if row < o and col < k else 0)
    again = wc.WideLinear8bit(n, k, o, bias=False)
    again.load_state_dict(mod.state_dict())
    assert torch.equal(again.dequantize(), want)


def test_linear8_from_modules():
    import wide_compiler as wc
    torch.manual_seed(1)
    mods = [torch.nn.Linear(70, 9) for _ in range(2)]
    with torch.no_grad():
        mods[0].weight[3] = 0
        mods[1].weight[2] *= 1e-41                          # codes under the smallest scale
        mods[1].weight[4] *= 1e30
    wide = wc.WideLinear8bit.from_modules(mods)
    w = torch.stack([m.weight for m in mods]).double()
    scale = (w.abs().amax(-1) / 127).clamp_min(2.0 ** -126)
    assert not ((wide.dequantize().double() - w).abs() > scale[..., None] * (0.5 + 2.0 ** -16)).any()
    assert torch.equal(wide.bias, torch.stack([m.bias for m in mods]))


def test_sampler_refusals(anywhere):
    import wide_compiler as wc
    for kw in (dict(temperature=[1.0, 2.0]), dict(temperature=-1.0), dict(top_p=float("nan")), dict(min_p=-0.1), dict(top_k=-1),
               dict(top_k=2.5), dict(top_k=1 << 31), dict(top_k=[1, 2, 3, 4])):
        with pytest.raises(ValueError):
            wc.WideSampler(3, **kw)
    s = wc.WideSampler(3, top_k=torch.tensor([1, 2, 3]), temperature=0.5)
    x, u = torch.zeros(3, 4, 9), torch.zeros(3, 4)
    with pytest.raises(AssertionError, match="launched"):
        s(x, u)
    for bad in ((x[:2], u[:2]), (x, u[:, :3]), (x, u.double()), (x, u.half()), (x[..., :0], u), (x[0, 0], u[0, 0]), (x, u[..., None])):
        with pytest.raises(RuntimeError):
            s(*bad)
    for kw in (dict(temperature=torch.ones(4).double()), dict(top_k=torch.ones(4).long()), dict(top_p=torch.ones(5)),
               dict(min_p=torch.ones(2, 3, 4))):
        with pytest.raises(RuntimeError):
            s(x, u, **kw)
    with pytest.raises(TypeError):
        s(x.double(), u)
    with pytest.raises(RuntimeError, match="forward-only"):
        s(x.requires_grad_(), u)


def test_sampler_rules(monkeypatch, anywhere):
    """What rules come to: their addresses and strides, in place when they change, the same after .to()."""
    import wide_compiler as wc
    from wide_compiler import _answer
    seen = []
    monkeypatch.setattr(_answer, "sample", lambda sizes, rows, need, x, u, rules, strides, tokens: seen.append((rules, strides)))
    s = wc.WideSampler(2, temperature=[0.5, 2.0], top_k=7, top_p=0.9, min_p=[0.1, 0.0])
    value = lambda i, t: s.rules[:, i].view(t).tolist() if t == torch.float32 else s.rules[:, i].tolist()  # noqa: E731
    assert s.rules[:, 0].contiguous().view(torch.float32).tolist() == [0.5, 2.0] and s.rules[:, 1].tolist() == [7, 7]
    at = s.rules.data_ptr()
    s.set(top_k=[0, 3])
    assert s.rules.data_ptr() == at and s.rules[:, 1].tolist() == [0, 3]
    before = s.rules.clone()
    assert torch.equal(s.to(torch.float16).rules, before)
    x, u = torch.zeros(2, 3, 5, 9), torch.zeros(2, 3, 5)
    given = torch.ones(3, 1)
    s(x, u, temperature=given, top_p=torch.ones(2, 3, 5), min_p=torch.ones(2, 5, 3).transpose(1, 2), top_k=torch.ones((), dtype=torch.int32))
    rules, strides = seen[0]
    assert strides == (15, 1, 0, 0, 15, 1, 15, 1)           # [3, 1] over [2, 3, 5] has two strides inside a model: copied
    s(x[:, :, 0], u[:, :, 0], temperature=given[:, 0])
    assert seen[1][0] == [given.data_ptr(), *(s.rules.data_ptr() + 4 * i for i in (1, 2, 3))]
    assert seen[1][1] == (0, 1, 4, 0, 4, 0, 4, 0)


def test_exports_are_refused(anywhere):
    import wide_compiler as wc
    pages = torch.zeros(5, 2, 16, 64)
    cache = wc.WidePagedCache.from_pages(pages, pages)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731

    class Calls(torch.nn.Module):
        def __init__(self, f):
            super().__init__()
            self.f = f

        def forward(self, x):
            return self.f(x)
    sampler, u = wc.WideSampler(1), torch.zeros(1, 2)
    for f, x in ((wc.WideLinear8bit(1, 64, 16), torch.zeros(1, 2, 64)), (lambda x: sampler(x, u), torch.zeros(1, 2, 64)),
                 (lambda x: cache.attend_shared(x, i(1, 1, 2), i(1, 1), i(1, 3, 4), i(1, 3)), torch.zeros(1, 3, 4, 64))):
        with torch.no_grad(), pytest.raises(RuntimeError, match="cannot be exported"):
            torch.export.export(Calls(f), (x,), strict=False)


def test_step_refuses_uneven_groups(anywhere):
    import wide_compiler as wc
    attn = wc.WideAttention(2, 128, 2).requires_grad_(False)
    pages = torch.zeros(5, 2, 16, 64)
    cache = wc.WidePagedCache.from_pages(pages, pages)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    for prefix, lens in (((i(2, 2, 4), i(2, 2)), i(2, 3)), ((i(2, 3, 4), i(1, 3)), i(2, 3)), ((i(2, 3, 4), i(2, 3)), i(2, 4)),
                         ((i(2, 0, 4), i(2, 0)), i(2, 3))):
        with pytest.raises(RuntimeError, match="groups of one size"):
            attn.step(torch.zeros(2, 3, 128), cache, i(2, 3, 4), lens, prefix=prefix)


def test_answer_host_side_clean_under_sanitizers():
    from tests.test_abi_sanitized import _asan_runtime
    if not os.path.exists(SAN_LIB) or _asan_runtime() is None:
        pytest.skip("the sanitizer-built library or its runtime is not there")
    env = dict(os.environ)
    env.update(LD_PRELOAD=_asan_runtime(), ASAN_OPTIONS="detect_leaks=0:abort_on_error=1:halt_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    probe = os.path.join(ROOT, "tests", "san_answer_probe.py")
    r = subprocess.run([sys.executable, probe, SAN_LIB, HEADER, "400", PKG], env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-6000:]
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr, r.stderr[-6000:]
    assert "no sanitizer report" in r.stdout


LINE = r"""
#include <cstdint>
#include <cstdio>
#include <vector>

#include "wc_shared.h"

// Units' tiles as one line in shares of shared_size tiles: units of none at all too, every tile in one share, no more shares
// than the budget, no two parts alike.
int main() {
  using namespace wc;
  uint32_t seed = 20261208;
  auto below = [&](int n) { return static_cast<int>((seed = seed * 1664525u + 1013904223u) >> 8) % n; };
  int none = 0;
  for (int it = 0; it < 50000; ++it) {
    const int units = 1 + below(below(2) ? 6 : 200), budget = 1 + below(below(2) ? 8 : 512), least = 1 + below(4), top = below(3) ? 1 + below(300) : 1;
    std::vector<int> tiles(units);
    int total = 0;
    for (int& t : tiles) total += t = below(top);
    const int size = shared_size(total, budget, least, units);
    if (size < 1) return 1;
    none += total == 0;
    if (total && (total - 1) / size + 1 > budget) return 2;
    std::vector<char> used(budget + units, 0);
    int start = 0;
    for (int s = 0; s < units; start += tiles[s++]) {
      const int first = start / size;
      for (int w = first; tiles[s] && w <= (start + tiles[s] - 1) / size; ++w) {
        if (w + s >= budget + units || used[w + s]) return 3;
        used[w + s] = 1;
      }
    }
  }
  printf("%d lines without tiles\n", none);
  return none > 100 ? 0 : 4;
}
"""


def test_shares_of_a_line_of_tiles(tmp_path):
    """How shared attention cuts its line of tiles, on the host, under the sanitizer that stops at a division by zero."""
    hipcc = next((h for h in ("/opt/rocm/bin/hipcc", "hipcc") if shutil.which(h)), None)
    if hipcc is None:
        pytest.skip("no hipcc")
    src, exe = tmp_path / "line.cpp", tmp_path / "line"
    src.write_text(LINE)
    r = subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-std=c++17", "-O1", "-w", "-Xarch_host", "-fsanitize=undefined", "-Xarch_host",
                        "-fno-sanitize-recover=undefined", "-I", os.path.join(PKG, "csrc"), "-I", os.path.join(ROOT, "include"), str(src),
                        "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr[-2000:])


FORM = r"""
#include <cstdio>
#include <cstdlib>

#include "wc_linear8.h"

int main(int argc, char** argv) {
  const char* names[] = {"fused", "few", "ring6", "ring3", "large", "tiles"};
  auto tiles = [](long x, long of) { return (x + of - 1) / of; };
  for (int i = 1; i + 3 < argc; i += 4) {
    const long n = atol(argv[i]), m = atol(argv[i + 1]), k = atol(argv[i + 2]), o = atol(argv[i + 3]);
    puts(names[static_cast<int>(wc::linear8_form(n, m, tiles(m, 16), tiles(o, 16), tiles(k, 128) * 2))]);
  }
}
"""


def test_the_tests_of_8_bit_products_reach_every_kernel(tmp_path):
    from tests.test_gpu_linear8bit import FORMS
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    src, exe = tmp_path / "form.cpp", tmp_path / "form"
    src.write_text(FORM)
    subprocess.run([gxx, "-std=c++17", "-I", os.path.join(PKG, "csrc"), str(src), "-o", str(exe)], check=True, timeout=120)
    shapes = [(form, shape) for form, each in FORMS.items() for shape in each]
    r = subprocess.run([str(exe), *(str(x) for _, shape in shapes for x in shape)], capture_output=True, text=True, timeout=60)
    assert r.stdout.split() == [form for form, _ in shapes], list(zip(r.stdout.split(), shapes))


def test_step_refuses_a_prefix_before_it_writes(anywhere, monkeypatch):
    import wide_compiler as wc

    def reached(*args, **kw):
        raise AssertionError("projected or written")
    attn = wc.WideAttention(2, 128, 2).requires_grad_(False)
    monkeypatch.setattr(attn, "_cached_heads", reached)
    pages = torch.zeros(5, 2, 16, 64)
    cache = wc.WidePagedCache.from_pages(pages, pages)
    monkeypatch.setattr(cache, "write", reached)
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(AssertionError, match="projected"):
        attn.step(torch.zeros(2, 4, 128), cache, i(2, 4, 1), i(2, 4), prefix=(i(2, 2, 4), i(2, 2)))
    for prefix in ((i(2, 2, 4).long(), i(2, 2)), (i(2, 2, 4), i(2, 2).long()), (i(2, 2), i(2, 2)), (i(2, 1, 4), i(2, 2)), (i(1, 2, 4), i(2, 2)),
                   (torch.zeros(2, 2, 4, dtype=torch.int32, device="meta"), i(2, 2))):
        with pytest.raises(RuntimeError, match="WideAttention.step"):
            attn.step(torch.zeros(2, 4, 128), cache, i(2, 4, 1), i(2, 4), prefix=prefix)


def test_sampler_rules_change_all_or_not_at_all():
    import wide_compiler as wc
    s = wc.WideSampler(2, temperature=0.7, top_k=5, top_p=0.9)
    before = s.rules.clone()
    for kw in (dict(temperature=2.0, top_k=-1), dict(temperature=1.0, top_p=[0.5, 0.5, 0.5]), dict(top_k=3, min_p=float("nan")),
               dict(top_k=float("inf")), dict(temperature=0.1, top_k=float("nan")), dict(top_p=0.1, min_p=-1.0)):
        with pytest.raises(ValueError):
            s.set(**kw)
        assert torch.equal(s.rules, before), kw
    s.set(temperature=float("inf"), top_k=[2 ** 31 - 1, 0])
    assert s.rules[:, 1].tolist() == [2 ** 31 - 1, 0]


def test_sampler_takes_an_empty_batch_with_rules_of_any_strides(anywhere):
    """Rules that a call copies, because a model's rows reach them by more than one stride, over batches without a row."""
    import wide_compiler as wc
    s = wc.WideSampler(2)
    for shape in ((2, 0, 5), (2, 5, 0), (2, 0)):
        for t in (torch.ones(()), torch.ones(shape[-1]), torch.ones(2, *[1] * (len(shape) - 1))):
            assert s(torch.zeros(*shape, 9), torch.zeros(shape), temperature=t).shape == shape
    none = wc.WideSampler(0)
    assert none(torch.zeros(0, 3, 5, 9), torch.zeros(0, 3, 5), top_p=torch.ones(3, 1)).shape == (0, 3, 5)


def test_linear8_keeps_the_largest_weight_finite():
    """fp32's largest value comes back as 127 of the largest scale whose 127 fp32 holds, a step of the scale less."""
    import wide_compiler as wc
    mod = torch.nn.Linear(5, 3)
    with torch.no_grad():
        mod.weight[1] = torch.finfo(torch.float32).max
        mod.weight[2, 0] = -torch.finfo(torch.float32).max
    back = wc.WideLinear8bit.from_modules([mod]).dequantize()[0]
    assert torch.isfinite(back).all()
    w = mod.weight.double()
    assert not ((back.double() - w).abs() > w.abs().amax(-1, keepdim=True) / 127 * (0.5 + 2.0 ** -15)).any()
