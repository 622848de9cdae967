"""The decode-step operators without a GPU: their header and binding agree, the library refuses bad arguments before any
launch, the modules refuse tensors they do not take, 4-bit weights pack and unpack exactly."""

import ctypes
import hashlib
import os
import re
import shutil
import struct
import subprocess
import sys
import tempfile

import pytest
import torch

from tests.conftest import PKG, ROOT
from tests._util import gen

HEADER = os.path.join(ROOT, "include", "wc_serve_abi.h")
SAN_LIB = os.path.join(PKG, "wide_compiler", "libwide_hip_san.so")


@pytest.fixture(scope="module")
def serve():
    from wide_compiler import _serve
    _serve.lib()
    return _serve


def _text():
    return re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)


def test_binding_declares_what_the_header_does(serve):
    declared = sorted(set(re.findall(r"\b(wc_[a-z0-9_]+)\s*\(", _text())))
    assert sorted(serve.SIGNATURES) == declared
    assert serve.lib().wc_serve_abi_version() == serve.ABI_VERSION
    # the fields of every struct, in order
    for cls, name in ((serve._HeadNormArgs, "wc_head_norm_args"), (serve._PagedCache, "wc_paged_cache"),
                      (serve._CacheWriteArgs, "wc_cache_write_args"), (serve._CacheReadArgs, "wc_cache_read_args"),
                      (serve._PagedAttnArgs, "wc_paged_attn_args"), (serve._Linear4Args, "wc_linear4_args")):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _text(), flags=re.S).group(1)
        fields = []
        for decl in body.split(";"):
            words = decl.replace("const", " ").replace("*", " ").split()
            if not words:
                continue
            if words[0] == "wc_paged_cache":
                fields += [f for f, _ in serve._PagedCache._fields_]
            else:
                fields += " ".join(words[1:]).replace(" ", "").split(",")
        assert [f for f, _ in cls._fields_] == fields, name


# a digest of include/wc_serve_abi.h without comments, per version
DECLARATIONS = {1: "e232a00a8c9af035227bbb304ee734af623bbc473e96d70fae216a89ac4b4811"}


def test_every_change_of_the_header_has_a_version_of_its_own(serve):
    assert DECLARATIONS.get(serve.ABI_VERSION) == hashlib.sha256(" ".join(_text().split()).encode()).hexdigest()


def _cache(a, **kw):
    for f, v in dict(dtype=1, bits=0, n=1, b=2, pages=4, page_size=16, heads=2, head_dim=64, row=64, k_pages=4096,
                     v_pages=4096, table=4096, table_len=3, table_stride=3, **kw).items():
        setattr(a, f, v)
    return a


def test_library_refuses_bad_arguments(serve):
    lib, big = serve.lib(), (1 << 63) - 1
    error = lambda: lib.wc_last_error().decode()  # noqa: E731
    for name, (_, args) in serve.SIGNATURES.items():
        if len(args) == 2:
            assert getattr(lib, name)(None, None) == -1, name
    assert lib.wc_paged_attention_workspace_bytes(None) == -1

    def norm(**kw):
        a = serve._HeadNormArgs()
        for f, v in dict(dtype=1, param_dtype=1, position_bytes=8, n=2, b=3, t=4, q_heads=4, k_heads=2, head_dim=64,
                         rotary_dim=64, q=4096, k=4096, q_out=4096, k_out=4096, q_weight=4096, k_weight=4096, freq=4096,
                         positions=4096, eps=1e-6, **{}).items():
            setattr(a, f, v)
        for f, v in kw.items():
            setattr(a, f, v)
        return lib.wc_head_norm_rotary(ctypes.byref(a), None)
    assert norm(dtype=5) == -3 and norm(position_bytes=2) == -3
    assert norm(head_dim=63) == -2 and norm(rotary_dim=66) == -2 and norm(rotary_dim=-2) == -2 and norm(b=-1) == -2
    assert norm(head_dim=258, rotary_dim=0) == -5 and norm(t=1 << 40) == -5 and norm(n=70000) == -5 and norm(q_heads=big) == -5
    assert norm(q=None) == -1 and norm(freq=None) == -1 and norm(q=4097) == -4 and norm(positions=4100) == -4
    assert norm(n=0) == 0 and norm(t=0) == 0

    def write(**kw):
        a = _cache(serve._CacheWriteArgs())
        a.t, a.k, a.v, a.start = 5, 4096, 4096, 4096
        for f, v in kw.items():
            setattr(a, f, v)
        return lib.wc_cache_write(ctypes.byref(a), None)
    assert write(dtype=9) == -3 and write(bits=4) == -3 and write(page_size=0) == -2 and write(row=60) == -2
    assert write(head_dim=300, row=512) == -5 and write(row=68) == -4 and write(pages=1 << 31) == -5 and write(b=big) == -5
    assert write(pages=1 << 20, page_size=1 << 12) == -5 and "2^31 rows" in error()
    assert write(k_pages=4104) == -4 and write(k_pages=None) == -1 and write(start=None) == -1 and write(k=4097) == -4
    assert write(bits=8) == -1 and write(t=big) == -5 and write(t=-1) == -2 and write(t=0) == 0 and write(b=0) == 0

    def read(**kw):
        a = _cache(serve._CacheReadArgs())
        a.lengths, a.max_length, a.k, a.v = 4096, 5, 4096, 4096
        for f, v in kw.items():
            setattr(a, f, v)
        return lib.wc_cache_read(ctypes.byref(a), None)
    assert read(max_length=-1) == -2 and read(max_length=big) == -5 and read(lengths=None) == -1 and read(v=4097) == -4
    assert read(max_length=0) == 0

    def attend(**kw):
        a = _cache(serve._PagedAttnArgs())
        a.q_heads, a.max_length, a.q, a.o, a.lengths, a.scale = 8, 4000, 4096, 4096, 4096, 0.1
        for f, v in kw.items():
            setattr(a, f, v)
        need = int(lib.wc_paged_attention_workspace_bytes(ctypes.byref(a)))
        return lib.wc_paged_attention(ctypes.byref(a), None), need
    assert attend(q_heads=3) == (-2, -1) and attend(q_heads=-2) == (-2, -1) and attend(max_length=-1) == (-2, -1)
    assert attend(max_length=big) == (-5, -1) and attend(q_heads=1 << 20) == (-5, -1) and attend(row=512, dtype=0) == (-5, -1)
    assert attend(q=None)[0] == -1 and attend(o=4097)[0] == -4 and attend(b=0) == (0, 0)
    # 4 key heads' worth of sequences split over their length need a workspace
    rc, need = attend(table_len=1000, max_length=16000)
    assert rc == -6 and need > 0 and "workspace" in error()
    assert attend(table_len=1000, max_length=16000, workspace=4100, workspace_bytes=need)[0] == -4
    assert attend(table_len=1000, max_length=16000, workspace=4096, workspace_bytes=need - 1)[0] == -6

    def linear(**kw):
        a = serve._Linear4Args()
        for f, v in dict(dtype=1, group=64, n=2, m=3, o=40, k=100, x=4096, x_rows_inner=3, codes=4096, scales=4096,
                         zeros=4096, y=4096).items():
            setattr(a, f, v)
        for f, v in kw.items():
            setattr(a, f, v)
        return lib.wc_linear4(ctypes.byref(a), None)
    assert linear(dtype=3) == -3 and linear(group=48) == -6 and linear(k=-1) == -2 and linear(k=0) == -2
    assert linear(o=big) == -5 and linear(k=big) == -5 and linear(x_rows_inner=1 << 32) == -5 and linear(x_rows_inner=0) == -6
    assert linear(codes=4100) == -4 and linear(scales=4104) == -4 and linear(x=4097) == -4 and linear(zeros=4097) == -4
    assert linear(y=None) == -1 and linear(m=0) == 0 and linear(o=0) == 0


def test_cpu_tensors_are_refused():
    import wide_compiler as wc
    for call in (lambda: wc.WideHeadNormRotary(1, 64)(torch.zeros(1, 1, 1, 2, 64), torch.zeros(1, 1, 1, 2, 64), torch.zeros(1).long()),
                 lambda: wc.WideLinear4bit(1, 64, 16)(torch.zeros(1, 2, 64)),
                 lambda: wc.WidePagedCache(2, 16, 2, 64, device="cpu"),
                 lambda: wc.WidePagedCache.from_pages(torch.zeros(2, 2, 16, 64), torch.zeros(2, 2, 16, 64))):
        with pytest.raises(RuntimeError, match="ROCm device tensors only"):
            call()


@pytest.fixture
def anywhere(monkeypatch):
    """Lets CPU tensors through the modules' checks, up to the launch, which must not be reached."""
    from wide_compiler import _hip, _serve

    def reached(*args, **kw):
        raise AssertionError("launched")
    monkeypatch.setattr(_hip, "require_device", lambda *a: None)
    for name in ("head_norm_rotary", "cache_write", "cache_read", "paged_attention", "linear4"):
        monkeypatch.setattr(_serve, name, reached)
    monkeypatch.setattr(_serve, "paged_attention_workspace", lambda *a: 0)


def test_head_norm_refusals(anywhere):
    import wide_compiler as wc
    for kw in (dict(head_dim=63), dict(head_dim=258), dict(head_dim=64, rotary_dim=66), dict(head_dim=64, rotary_dim=5), dict(head_dim=0)):
        with pytest.raises(ValueError):
            wc.WideHeadNormRotary(2, **kw)
    with pytest.raises(ValueError):
        wc.WideHeadNormRotary.from_modules([torch.nn.RMSNorm(64)], [torch.nn.RMSNorm(64), torch.nn.RMSNorm(64)])
    with pytest.raises(ValueError):
        wc.WideHeadNormRotary.from_modules([torch.nn.RMSNorm(64)], [torch.nn.RMSNorm(32)])
    mod = wc.WideHeadNormRotary(2, 64).requires_grad_(False)
    q, k, pos = torch.zeros(2, 3, 4, 6, 64), torch.zeros(2, 3, 4, 2, 64), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(AssertionError, match="launched"):
        mod(q, k, pos)
    for args in ((q[:1], k, pos), (q[..., :32], k, pos), (q, k[:, :2], pos), (q, k.half(), pos), (q, k, pos.float()),
                 (q, k, torch.zeros(5, dtype=torch.int64)), (q[0], k, pos), (q, k, torch.zeros(1, 2, 3, 4, dtype=torch.int64)),
                 (q.double(), k.double(), pos)):
        with pytest.raises((RuntimeError, TypeError)):
            if args[0].dtype == torch.float64:
                from wide_compiler import _hip
                _hip.dtype_code(args[0].dtype, "head_norm")
            mod(*args)
    with pytest.raises(RuntimeError, match="forward-only"):
        mod(q.requires_grad_(), k, pos)


def test_cache_refusals(anywhere):
    import wide_compiler as wc
    pages = torch.zeros(5, 2, 16, 64, dtype=torch.bfloat16)
    i8, scales = torch.zeros(5, 2, 16, 64, dtype=torch.int8), torch.zeros(5, 2, 16)
    f = wc.WidePagedCache.from_pages
    for args, kw in (((pages, pages[:4]), {}), ((pages, pages.half()), {}), ((pages, pages), dict(dtype=torch.float16)),
                     ((pages, pages, scales, scales), {}), ((i8, i8), dict(dtype=torch.bfloat16)),
                     ((i8, i8, scales, scales.half()), dict(dtype=torch.bfloat16)),
                     ((i8, i8, scales, scales[:4]), dict(dtype=torch.bfloat16)),
                     ((pages, pages), dict(head_dim=65)), ((pages, pages), dict(head_dim=0)),
                     ((pages[..., :60].contiguous(), pages[..., :60].contiguous()), {}),
                     ((pages.transpose(1, 2), pages.transpose(1, 2)), {}), ((pages[:, :, :0], pages[:, :, :0]), {}),
                     ((i8, i8, scales, None), dict(dtype=torch.bfloat16)), ((pages[:, :0], pages[:, :0]), {})):
        with pytest.raises(ValueError):
            f(*args, **kw)
    with pytest.raises(TypeError):
        f(pages.double(), pages.double())
    with pytest.raises(TypeError):
        f(i8, i8, scales, scales)                            # of which dtype?
    with pytest.raises(ValueError):
        wc.WidePagedCache(2, 16, 2, 300, device="cpu")
    cache = f(pages, pages)
    k = torch.zeros(1, 3, 7, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(1, 3, 4, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 3, 4, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32)
    for call in (lambda: cache.write(k, k, table, n), lambda: cache.read(table, n, 9), lambda: cache.attend(q, table, n)):
        with pytest.raises(AssertionError, match="launched"):
            call()
    for call in (lambda: cache.write(k[..., :32], k[..., :32], table, n), lambda: cache.write(k, k[:, :, :6], table, n),
                 lambda: cache.write(k.half(), k.half(), table, n), lambda: cache.write(k, k, table.long(), n),
                 lambda: cache.write(k, k, table[:, :2], n), lambda: cache.write(k, k, table, n.long()),
                 lambda: cache.write(k, k, table, n[:, :2]), lambda: cache.write(k, k, table, n, n.float()),
                 lambda: cache.write(k[:, :, :, :1], k[:, :, :, :1], table, n), lambda: cache.read(table[0], n, 9),
                 lambda: cache.read(table, n, -1), lambda: cache.read(table, n[0], 9),
                 lambda: cache.attend(q[..., :32], table, n), lambda: cache.attend(q[:, :, :3], table, n),
                 lambda: cache.attend(q.half(), table, n), lambda: cache.attend(q, table, n, first=n[:, :1]),
                 lambda: cache.attend(q, table, n, max_length=-1), lambda: cache.attend(q[None], table, n)):
        with pytest.raises(RuntimeError):
            call()


def test_linear4_refusals(anywhere):
    import wide_compiler as wc
    for args, kw in (((1, 64, 16), dict(group_size=48)), ((1, 0, 16), {})):
        with pytest.raises(ValueError):
            wc.WideLinear4bit(*args, **kw)
    with pytest.raises(TypeError):
        wc.WideLinear4bit(1, 64, 16, dtype=torch.float64)
    codes, scales = torch.zeros(2, 16, 32, dtype=torch.uint8), torch.ones(2, 16, 1)
    zeros = torch.zeros(2, 16, 1, dtype=torch.uint8)
    f = wc.WideLinear4bit.from_codes
    for kw in (dict(codes=codes.int()), dict(codes=codes[0]), dict(in_features=66), dict(scales=scales[:, :8]),
               dict(zeros=zeros + 16), dict(zeros=zeros.int()), dict(bias=torch.zeros(2, 15)), dict(group_size=32),
               dict(group_size=0)):
        kw = dict(codes=codes, scales=scales, in_features=64, group_size=64, zeros=zeros) | kw
        with pytest.raises(ValueError):
            f(kw.pop("codes"), kw.pop("scales"), **kw)
    mod = f(codes, scales, in_features=64, group_size=64, zeros=zeros)
    with pytest.raises(AssertionError, match="launched"):
        mod(torch.zeros(2, 3, 64))
    for x in (torch.zeros(2, 3, 32), torch.zeros(1, 3, 64), torch.zeros(2, 3, 64).half(), torch.zeros(64)):
        with pytest.raises(RuntimeError):
            mod(x)
    # buffers that were replaced since the last call
    x = torch.zeros(2, 3, 64)
    for name, t in (("packed", mod.packed[:, :, :, :32]), ("packed", mod.packed.long()), ("scales", mod.scales[..., :8]),
                    ("zeros", mod.zeros[:1]), ("zeros", mod.zeros.int()), ("bias", torch.zeros(2, 15))):
        old = getattr(mod, name)
        setattr(mod, name, t)
        with pytest.raises(RuntimeError, match=name):
            mod(x)
        setattr(mod, name, old)
    with pytest.raises(AssertionError, match="launched"):
        mod(x)


@pytest.mark.parametrize("n,o,k,group,zeros", [(2, 500, 1000, 32, True), (1, 16, 128, 128, False), (3, 5, 37, 64, True),
                                               (1, 33, 129, 32, False), (2, 1, 1, 128, True)])
def test_linear4_codes_pack_and_unpack_exactly(n, o, k, group, zeros):
    import wide_compiler as wc
    g = gen(k)
    codes = torch.randint(0, 256, (n, o, (k + 1) // 2), generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    scales = torch.rand(n, o, groups, generator=g)
    z = torch.randint(0, 16, (n, o, groups), generator=g, dtype=torch.uint8) if zeros else None
    mod = wc.WideLinear4bit.from_codes(codes, scales, in_features=k, group_size=group, zeros=z)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)[..., :k].float()
    at = torch.arange(k) // group
    assert torch.equal(mod.dequantize(), (c - (z.float()[..., at] if zeros else 8.0)) * scales[..., at])


def test_serve_host_side_clean_under_sanitizers():
    from tests.test_abi_sanitized import _asan_runtime
    if not os.path.exists(SAN_LIB) or _asan_runtime() is None:
        pytest.skip("the sanitizer-built library or its runtime is not there")
    env = dict(os.environ)
    env.update(LD_PRELOAD=_asan_runtime(), ASAN_OPTIONS="detect_leaks=0:abort_on_error=1:halt_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    probe = os.path.join(ROOT, "tests", "san_serve_probe.py")
    r = subprocess.run([sys.executable, probe, SAN_LIB, HEADER, "400", PKG], env=env, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr[-6000:]
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr, r.stderr[-6000:]
    assert "no sanitizer report" in r.stdout


COUNT = r"""
#include <cstdio>
#include <cstdlib>

#include "wc_paged.h"

// What the attention kernel counts in 32 bits (the tiles of all sequences, a share's end), here in 64 beside it, for lengths
// that say anything: none may differ, and a share's parts are at most the shares.
int main() {
  using namespace wc;
  srand(20261206);
  const int64_t extreme = (1ll << 31) - 65, budgets[] = {1, 7, 256, 768, 1024};
  const int32_t garbage[] = {2147483647, 2147483583, 2147483640, 1 << 30, -1, 1025, 0, 100, 1048577};
  int cut = 0, counted = 0;
  for (int it = 0; it < 20000; ++it) {
    wc_paged_cache c = {};
    c.pages = rand() % 8 ? 4 : 0;
    c.page_size = 1ll << rand() % 25;
    c.table_len = rand() % 3 ? rand() % 4096 : extreme;
    const int64_t seqs = 1 + rand() % (rand() % 2 ? 2047 : 40), budget = budgets[rand() % 5];
    const int64_t max_length = rand() % 3 ? extreme : rand() % 4096, most = paged_most(c, max_length);
    if (most > max_length || most > c.table_len * c.page_size || (!c.pages && most)) return 1;
    if (!paged_countable(seqs, most)) continue;
    int64_t total = 0;
    uint32_t total32 = 0;                                  // as the kernel adds, without undefined overflow here
    for (int64_t s = 0; s < seqs; ++s) {
      const int32_t length = garbage[rand() % 9], first = rand() % 2 ? 0 : garbage[rand() % 9];
      const PagedSpan span = paged_span(first, length, static_cast<int32_t>(most));
      if (span.hi > most || span.lo < 0 || span.cut != (length > most)) return 2;
      const int64_t lo = span.lo / 32 * 32, want = span.hi > span.lo ? (span.hi - lo + 31) / 32 : 0;
      if (paged_tiles(span) != want) return 3;
      cut += span.cut;
      total += want;
      total32 += static_cast<uint32_t>(paged_tiles(span));
    }
    const int64_t size = std::max<int64_t>((total + budget - 1) / budget, 8);
    if (total != static_cast<int32_t>(total32) || (budget - 1) * size + size > 2147483647ll + 8 * 1024 || total + size > 2147483647ll) return 4;
    if (total && (total - 1) / size + 1 > budget) return 5;
    ++counted;
  }
  printf("%d counted, %d cut\n", counted, cut);
  return counted > 1000 && cut > 1000 ? 0 : 6;
}
"""


def test_attention_counts_tiles_within_32_bits(tmp_path):
    """The bound of a sequence's tokens is the one that the count of all tiles is checked with: neither lengths that say
    anything nor a max_length far over what the tables name take the line of tiles, its shares or a join's parts out of
    their range."""
    hipcc = next((h for h in ("/opt/rocm/bin/hipcc", "hipcc") if shutil.which(h)), None)
    if hipcc is None:
        pytest.skip("no hipcc")
    src, exe = tmp_path / "count.cpp", tmp_path / "count"
    src.write_text(COUNT)
    r = subprocess.run([hipcc, "-x", "hip", "--offload-host-only", "-std=c++17", "-O1", "-w", "-I", os.path.join(PKG, "csrc"), "-I",
                        os.path.join(ROOT, "include"), str(src), "-o", str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-4000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, (r.returncode, r.stdout)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("eps", [None, 1e-5])
def test_head_norm_from_modules_has_the_eps_that_rms_norm_uses(eps, dtype):
    """Rows as small as eps: what nn.RMSNorm gives (up to its roundings of the norm, the weight's product and the sum:
    4 steps) is the formula with the converted module's eps."""
    import wide_compiler as wc
    norm = torch.nn.RMSNorm(96, eps=eps).to(dtype)
    mod = wc.WideHeadNormRotary.from_modules([norm], [norm])
    for size in (1.0, 1e-2, 1e-3):
        x = (size * torch.randn(50, 96, generator=gen(3))).to(dtype)
        ref = x.double() / (x.double().square().mean(-1, keepdim=True) + mod.eps).sqrt()
        step = torch.finfo(dtype).eps
        with torch.no_grad():
            assert ((norm(x).double() - ref).abs() <= 4 * step * ref.abs() + 4 * torch.finfo(dtype).tiny * step + 100 * 2.0 ** -24 * ref.abs()).all()


def test_head_norm_from_modules_of_norms_with_and_without_weights():
    """The type is that of the weights there are, wherever they stand; norms of several types are refused."""
    import wide_compiler as wc
    plain, own = torch.nn.RMSNorm(32, elementwise_affine=False), torch.nn.RMSNorm(32, dtype=torch.bfloat16)
    torch.nn.init.normal_(own.weight)
    mod = wc.WideHeadNormRotary.from_modules([plain, plain], [own, plain])
    assert mod.k_weight.dtype == mod.q_weight.dtype == torch.bfloat16
    assert torch.equal(mod.k_weight[0], own.weight) and (mod.k_weight[1] == 1).all() and (mod.q_weight == 1).all()
    assert wc.WideHeadNormRotary.from_modules([plain], [plain]).q_weight.dtype == torch.float32
    with pytest.raises(ValueError, match="one dtype"):
        wc.WideHeadNormRotary.from_modules([own], [torch.nn.RMSNorm(32)])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1.0, 1e-3, 3e-4, 3e-5, 1e-6, 6e-8, 2e-38, 0.0])
@pytest.mark.parametrize("group", [32, 128])
def test_linear4_from_modules_spans_small_weights(group, size, dtype):
    """Codes span a group's values at any size that the type has: a value is off by half of the stored scale s, or, at the
    upper end, by s / 2 and what s is under (max - min) / 15 (at most half a rounding step of it, 15 times); s is at most
    that step's rounding, or up to the type's smallest value more."""
    import wide_compiler as wc
    torch.manual_seed(5)
    lin = [torch.nn.Linear(150, 40, bias=False).to(dtype) for _ in range(2)]
    for m in lin:
        torch.nn.init.uniform_(m.weight, -size, size)
        m.weight.data[3] = m.weight.data[3].abs()             # a row of one sign
        m.weight.data[4] = 0
    mod = wc.WideLinear4bit.from_modules(lin, group_size=group)
    groups = -(-150 // group)
    w = torch.stack([m.weight for m in lin]).detach().double()
    pad = torch.nn.functional.pad(w, (0, groups * group - 150)).unflatten(-1, (groups, group))
    step = (pad.amax(-1).clamp_min(0) - pad.amin(-1).clamp_max(0)) / 15
    s = mod.scales.transpose(2, 3).reshape(2, -1, mod.scales.shape[2])[:, :40, :groups].double()
    info = torch.finfo(dtype)
    off = (torch.nn.functional.pad(mod.dequantize().double() - w, (0, groups * group - 150))).unflatten(-1, pad.shape[2:]).abs().amax(-1)
    assert (off <= s * (0.5 + 8 * info.eps + 1e-5)).where(step > 0, off == 0).all()
    assert (s <= step * (1 + info.eps) + info.tiny * info.eps).where(step > 0, s > 0).all()


def test_linear4_from_modules_of_several_kinds_are_refused():
    """A bias would be lost, a type rounded, where only the first module were looked at."""
    import wide_compiler as wc
    lin = torch.nn.Linear
    for a, b in ((lin(64, 16, bias=False), lin(64, 16)), (lin(64, 16), lin(64, 16, bias=False)), (lin(64, 16), lin(64, 17)),
                 (lin(64, 16), lin(32, 16)), (lin(64, 16).half(), lin(64, 16))):
        with pytest.raises(ValueError, match="one shape, dtype and device"):
            wc.WideLinear4bit.from_modules([a, b], group_size=32)


def test_head_norm_rotation_is_fixed(monkeypatch, anywhere):
    """A call's plan and the frequencies are made from the rotation's numbers: they cannot be set apart from them.  eps,
    which every call reads, can."""
    import wide_compiler as wc
    from wide_compiler import _serve
    mod = wc.WideHeadNormRotary(1, 64, rotary_dim=32, base=500.0, interleaved=True).requires_grad_(False)
    assert (mod.rotary_dim, mod.base, mod.interleaved) == (32, 500.0, True)
    for name, value in (("rotary_dim", 64), ("base", 10000.0), ("interleaved", False)):
        with pytest.raises(AttributeError):
            setattr(mod, name, value)
    seen = []
    monkeypatch.setattr(_serve, "head_norm_rotary", lambda plan, *a: seen.append((plan[0][2], plan[0][10], a[-1])))
    q, pos = torch.zeros(1, 1, 2, 3, 64), torch.zeros(2, dtype=torch.int64)
    mod(q, q, pos)
    mod.eps = 1e-3
    mod(q, q, pos)
    assert seen == [(1, 32, 1e-6), (1, 32, 1e-3)]


def test_exports_are_refused(anywhere):
    """torch.export traces through what torch.compile steps out of: an error that says so, not a recursion."""
    import wide_compiler as wc
    pages = torch.zeros(5, 2, 16, 64)
    cache = wc.WidePagedCache.from_pages(pages, pages)
    table, n = torch.zeros(1, 3, 4, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32)
    k, q = torch.zeros(1, 3, 7, 2, 64), torch.zeros(1, 3, 4, 64)

    class Calls(torch.nn.Module):
        def __init__(self, f):
            super().__init__()
            self.f = f

        def forward(self, x):
            return self.f(x)
    norm = wc.WideHeadNormRotary(1, 64).requires_grad_(False)
    for f, x in ((wc.WideLinear4bit(1, 64, 16), torch.zeros(1, 2, 64)), (lambda x: norm(x, x, n[0, 0]), k),
                 (lambda x: cache.attend(x, table, n), q), (lambda x: cache.write(x, x, table, n), k),
                 (lambda x: cache.read(table, n, 4), k)):
        with torch.no_grad(), pytest.raises(RuntimeError, match="cannot be exported"):
            torch.export.export(Calls(f), (x,), strict=False)


def test_parametrised_weights_count(monkeypatch, anywhere):
    """A weight or scale that torch parametrises, or a bias that became a parameter, is read as any other module reads it."""
    import wide_compiler as wc
    from torch.nn.utils import parametrize
    from wide_compiler import _serve

    class Twice(torch.nn.Module):
        def forward(self, w):
            return 2 * w
    seen = []
    monkeypatch.setattr(_serve, "head_norm_rotary", lambda plan, q, k, qo, ko, qw, kw, *a: seen.append((qw, kw)))
    monkeypatch.setattr(_serve, "linear4", lambda sizes, rows, x, codes, scales, zeros, bias, y: seen.append((scales, bias)))
    norm = wc.WideHeadNormRotary(1, 64)
    parametrize.register_parametrization(norm, "k_weight", Twice())
    lin = wc.WideLinear4bit(1, 64, 16, group_size=64)
    lin.scales.fill_(1)
    parametrize.register_parametrization(lin, "scales", Twice())
    del lin.bias
    lin.bias = torch.nn.Parameter(torch.ones(1, 16))
    q = torch.zeros(1, 1, 2, 3, 64)
    with torch.no_grad():
        norm(q, q, torch.zeros(2, dtype=torch.int64))
        lin(torch.zeros(1, 2, 64))
    (qw, kw), (scales, bias) = seen
    assert (qw == 1).all() and (kw == 2).all() and (scales == 2).all() and (bias == 1).all()
    with pytest.raises(RuntimeError, match="forward-only"):
        lin(torch.zeros(1, 2, 64))                          # its bias asks for a gradient


def test_a_growing_bound_keeps_the_plans(monkeypatch, anywhere):
    """max_length raised with every token, as a tight bound is: the call's form stays checked, and no other form's plan is
    lost to it."""
    import wide_compiler as wc
    from wide_compiler import _serve
    for name in ("cache_write", "cache_read", "paged_attention"):
        monkeypatch.setattr(_serve, name, lambda *a: None)
    pages = torch.zeros(5, 2, 16, 64)
    cache = wc.WidePagedCache.from_pages(pages, pages)
    table, n = torch.zeros(1, 3, 4, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32)
    k, q = torch.zeros(1, 3, 7, 2, 64), torch.zeros(1, 3, 4, 64)
    cache.write(k, k, table, n)
    checked = []
    monkeypatch.setattr(wc.WidePagedCache, "_check_table", staticmethod(lambda *a: checked.append(a)))
    for length in range(1000):
        cache.attend(q, table, n, max_length=length)
        assert cache.read(table, n, length % 9)[0].shape == (1, 3, length % 9, 2, 64)
    cache.write(k, k, table, n)
    assert len(checked) == 2                                 # the first attend and the first read
    for call in (lambda: cache.attend(q, table, n, max_length=-1), lambda: cache.read(table, n, -1)):
        with pytest.raises(RuntimeError, match="negative"):
            call()


def test_head_norm_made_on_the_meta_device_turns_as_any_other():
    """Frequencies are no part of a state_dict: a module that gets its memory later has them all the same."""
    import wide_compiler as wc
    made = wc.WideHeadNormRotary(2, 64, rotary_dim=32, base=500.0)
    with torch.device("meta"):
        later = wc.WideHeadNormRotary(2, 64, rotary_dim=32, base=500.0)
    assert later._freq_bits.is_meta and later.half()._freq_bits.is_meta
    torch.full((16,), 7)                                     # what to_empty may find in memory
    later = later.to_empty(device="cpu")
    later.load_state_dict(made.state_dict(), strict=True)
    assert torch.equal(later._freq_bits, made._freq_bits) and later._freq_bits.view(torch.float64)[0] > 0.1
    assert torch.equal(made.to(torch.bfloat16)._freq_bits, later._freq_bits)
    none = wc.WideHeadNormRotary(1, 64, rotary_dim=0).double()
    assert none._freq_bits.numel() == 0


def _kernel_registers(part):
    """{mangled name: (VGPRs with AGPRs, bytes of scratch)} of the kernels in the built library whose name has `part`: what
    the compiler wrote into the notes of its code objects."""
    readelf = next((r for r in ("/opt/rocm/llvm/bin/llvm-readelf", "llvm-readelf") if shutil.which(r)), None)
    if readelf is None:
        pytest.skip("no llvm-readelf")
    data = open(os.path.join(PKG, "wide_compiler", "libwide_hip.so"), "rb").read()
    magic, found, at = b"__CLANG_OFFLOAD_BUNDLE__", {}, -1
    while (at := data.find(magic, at + 1)) >= 0:
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            target = data[entry + 24:entry + 24 + length]
            entry += 24 + length
            code = data[at + offset:at + offset + size]
            if b"gfx950" not in target or part.encode() not in code:
                continue
            with tempfile.NamedTemporaryFile() as f:
                f.write(code)
                f.flush()
                notes = subprocess.run([readelf, "--notes", f.name], capture_output=True, text=True, timeout=60).stdout
            for kernel in notes.split("  - .agpr_count:")[1:]:
                field = lambda name: re.search(r"\.%s:\s+(\S+)" % name, kernel).group(1)  # noqa: E731
                if part in field("symbol"):
                    found[field("symbol")] = (int(field("vgpr_count")), int(field("private_segment_fixed_size")))
    return found


def test_attention_shares_follow_the_registers():
    """The number of workgroups a compute unit has room for, by which paged attention cuts its line of tiles, is what the
    built kernels' registers leave: of 512 a lane and quarter of a unit, in steps of 8, for workgroups of a wave each."""
    source = open(os.path.join(PKG, "csrc", "paged_attention.hip")).read()
    fit = re.search(r"kFit\[2\]\[3\]\[3\] = \{(.*)\};", source).group(1)
    fit = [int(x) for x in re.findall(r"\d+", fit)]
    kernels = _kernel_registers("paged_attention_kernel")
    seen = 0
    for q8 in (0, 1):
        for t, name in enumerate(("f", "DF16b", "DF16_")):
            for w, dc in enumerate((64, 128, 256)):
                stored = "a" if q8 else "S3_" if name != "f" else "f"
                match = [k for k in kernels if re.search(r"kernelI%s(%s|%s)Li%dELi4E" % (name, stored, "a" if q8 else name, dc), k)]
                assert len(match) == 1, (name, q8, dc, match)
                registers = -(-kernels[match[0]][0] // 8) * 8
                assert fit[(q8 * 3 + t) * 3 + w] == min(512 // registers, 8), (match[0], registers)
                seen += 1
    assert seen == 18
