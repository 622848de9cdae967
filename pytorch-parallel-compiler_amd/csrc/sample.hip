// Draws a token of every row of logits by temperature, top-k, top-p and min-p, from a given random number.
//
//   w_i = exp((x_i - max x) / t);  kept: the first of the order (value down, index up);  the token is the lowest kept
//   index up to which the kept weights pass u times their sum
//
// The filters all keep the first of one order, so a kept set is a border: a value T, all above it and the first q
// of those equal to it.  It is found on the values' bits as ordered integers, bin by bin: counts and weights of the
// bins of a range, then of the bins inside the bin where the border falls.
//
// Which token comes out must not hang on the order of a sum, so weights are summed as whole numbers, of 2^-48 of the
// largest weight (more where rows are so long that 64 bits could not hold the sum): each is the exponential in 64 bits,
// off by 2^-46 of itself, and rounded once, to 1 at least, so that u = 0 gives the first that has a weight at all.
#include <algorithm>

#include "wc_answer_abi.h"
#include "wc_common.h"

namespace wc {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;

struct Sample {
  const char* x;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int64_t* tokens;
  int64_t xn, xo, xi, tn, tm, kn, km, pn, pm, mn, mm;
  int32_t v, fraction;       // fraction: bits below the largest weight that sums hold
  FastDiv by_m, by_rows;
};

// A value as an integer of the same order; NaN is -infinity, zeros are one value.
constexpr uint32_t kNever = 0x007fffffu;             // -infinity
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return x == x ? k : kNever;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Weights as whole numbers: 2^(y + fraction), y = (x - max) log2(e) / t, with 2^(i/64) from a table and the rest, at most
// 2^-7 of a power, from the first terms of its series, whose next is under 2^-58.
struct Weights {
  const double* table;       // 64
  double most, scale;
  float top;
  int fraction;
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (!(x > -INFINITY)) return 0;
    // + 0: where x and max are the same infinity, or t is infinite
    double y = x == top ? 0.0 : (static_cast<double>(x) - most) * scale;
    if (!(y > -1075.0)) return 0;                    // under what 64 bits hold
    constexpr double magic = 0x1.8p52;
    const double n = fma(y, 64.0, magic);
    const int i = static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, n)));
    const double f = fma(y, 64.0, magic - n);
    constexpr double l = 0.69314718055994530942 / 64;
    double p = l * l * l * l * l / 120;
    p = fma(p, f, l * l * l * l / 24);
    p = fma(p, f, l * l * l / 6);
    p = fma(p, f, l * l / 2);
    p = fma(p, f, l);
    p = fma(p, f, 1.0);
    p = ldexp(p * table[i & 63], (i >> 6) + fraction);
    return max(__builtin_bit_cast(uint64_t, p + 0x1p52) - __builtin_bit_cast(uint64_t, 0x1p52), static_cast<uint64_t>(1));
  }
};

// The border of a kept set: all keys above `key`, and the first `ties` of those that are it.
struct Border {
  uint32_t key;
  uint32_t ties;
};

struct Shared {
  uint64_t weight[kBins];
  uint32_t count[kBins];
  double table[64];
  uint64_t wave64[kWaves];
  uint32_t wave32[kWaves];
  uint64_t found64[2];
  uint32_t found32[4];
};

template <typename T>
struct Row {
  static constexpr int E = 16 / sizeof(T);
  const T* x;
  int v;
  // go(value, index) for the values from 16 bytes times `piece` on
  template <typename F>
  __device__ __forceinline__ void piece(int64_t at, F go) const {
    if (at + E <= v) {
      T t[E];
      __builtin_memcpy(t, x + at, 16);               // at element alignment
#pragma unroll
      for (int e = 0; e < E; ++e) go(to_f32(t[e]), static_cast<int>(at) + e);
    } else {
      for (int64_t i = at; i < v; ++i) go(to_f32(x[i]), static_cast<int>(i));
    }
  }
  template <typename F>
  __device__ __forceinline__ void all(F go) const {
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * E; at < v; at += kThreads * E) piece(at, go);
  }
};

// sums over the workgroup of values of all lanes before this one, and of all of them
__device__ __forceinline__ uint64_t before64(uint64_t v, Shared& s, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t sum = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t up = __shfl_up(static_cast<unsigned long long>(sum), off, 64);
    if (lane >= off) sum += up;
  }
  __syncthreads();
  if (lane == 63) s.wave64[wave] = sum;
  __syncthreads();
  uint64_t base = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) base += s.wave64[w];
    total += s.wave64[w];
  }
  return base + sum - v;
}

// The border at which what is kept from the top first reaches `limit`, of counts (COUNT) or of weights; limit > 0 and at
// most what all keys above kNever have.  Keys above `from` count, and the first `ties` of those that are it.
template <bool COUNT, typename T>
__device__ Border find_border(const Row<T>& row, const Weights& w, Shared& s, uint32_t top, Border from, uint64_t limit) {
  uint32_t lo = max(from.key, kNever + 1), hi = top;
  uint64_t above = 0;
  for (;;) {
    const uint32_t width = hi - lo;
    const int shift = max(0, 32 - __clz(width | 1) - 11);          // bins of 2^shift keys, at most kBins
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.weight[i] = 0;
      s.count[i] = 0;
    }
    __syncthreads();
    row.all([&](float x, int) {
      const uint32_t k = key_of(x);
      if (k < lo || k > hi) return;
      const uint32_t b = (k - lo) >> shift;
      atomicAdd(&s.count[b], 1u);
      if (!COUNT) atomicAdd(reinterpret_cast<unsigned long long*>(&s.weight[b]), static_cast<unsigned long long>(w(x)));
    });
    __syncthreads();
    // ties of `from` that don't count
    if (threadIdx.x == 0 && lo == from.key && s.count[0] > from.ties && shift == 0) {
      s.weight[0] = COUNT ? 0 : s.weight[0] / s.count[0] * from.ties;
      s.count[0] = from.ties;
    }
    __syncthreads();
    // bins from the top, two a thread
    const int b1 = kBins - 1 - 2 * threadIdx.x, b0 = b1 - 1;
    const uint64_t v1 = COUNT ? s.count[b1] : s.weight[b1], v0 = COUNT ? s.count[b0] : s.weight[b0];
    uint64_t total;
    const uint64_t start = above + before64(v1 + v0, s, total);
    if (start < limit && start + v1 + v0 >= limit) {
      const bool first = start + v1 >= limit;
      s.found32[0] = first ? b1 : b0;
      s.found64[0] = first ? start : start + v1;
    }
    __syncthreads();
    const uint32_t bin = s.found32[0];
    above = s.found64[0];
    lo += bin << shift;
    if (shift == 0) {
      const uint64_t left = limit - above, have = s.count[bin];
      const uint64_t each = COUNT ? 1 : s.weight[bin] / have;
      return Border{lo, static_cast<uint32_t>(min((left + each - 1) / each, have))};
    }
    hi = min(hi, lo + ((1u << shift) - 1));
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(Sample a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t model = fdiv(blockIdx.x, a.by_m), r = blockIdx.x - model * a.by_m.d, outer = fdiv(r, a.by_rows);
  const Row<T> row{reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (r - outer * a.by_rows.d) * a.xi, a.v};
  const float t = a.temperature[model * a.tn + r * a.tm], top_p = a.top_p[model * a.pn + r * a.pm];
  const float min_p = a.min_p[model * a.mn + r * a.mm], u = a.u[blockIdx.x];
  const int32_t top_k = a.top_k[model * a.kn + r * a.km];
  if (tid < 64) s.table[tid] = exp2(tid / 64.0);

  // the first of the order: the largest key, then the lowest index
  uint64_t best = 0;
  row.all([&](float x, int i) { best = max(best, static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~i)); });
#pragma unroll
  for (int off = 32; off; off >>= 1) best = max(best, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best), off, 64)));
  if (lane == 0) s.wave64[wave] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) best = max(best, s.wave64[w]);
  const uint32_t top = best >> 32;
  const int first = static_cast<int>(~static_cast<uint32_t>(best));
  if (top <= kNever || !(t > 0.f) || top_k == 1 || top_p <= 0.f) {
    if (tid == 0) a.tokens[blockIdx.x] = top <= kNever ? -1 : first;
    return;
  }
  const float most = value_of(top);
  const Weights w{s.table, most, 1.4426950408889634074 / t, most, a.fraction};

  // the border, and the least weight
  Border border{kNever, 0};
  if (top_k > 0 && top_k < a.v) {
    // no more than there are above -infinity: counted by the way, as bins' totals
    uint64_t total;
    uint32_t mine = 0;
    row.all([&](float x, int) { mine += key_of(x) > kNever; });
    before64(mine, s, total);
    if (static_cast<uint64_t>(top_k) < total) border = find_border<true>(row, w, s, top, border, top_k);
  }
  // kept by the border, ties in doubt counted apart
  auto weight = [&](float x, uint32_t& ties) {
    const uint32_t k = key_of(x);
    ties += k == border.key && border.ties;
    return k > border.key ? w(x) : 0;
  };
  if (top_p < 1.f) {
    uint64_t sum = 0, total;
    uint32_t ties = 0;
    row.all([&](float x, int) { sum += weight(x, ties); });
    before64(sum, s, total);
    if (border.ties) total += border.ties * w(value_of(border.key));
    const double part = static_cast<double>(top_p) * static_cast<double>(total);
    const uint64_t limit = max(static_cast<uint64_t>(ceil(part)), static_cast<uint64_t>(1));
    border = find_border<false>(row, w, s, top, border, min(limit, total));
  }
  if (min_p > 0.f) {
    // the least key whose weight reaches min_p: found by halves
    uint32_t lo = border.key, hi = top;              // hi reaches it
    const double least = ldexp(static_cast<double>(fminf(min_p, 1.f)), a.fraction);
    while (lo + 1 < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (static_cast<double>(w(value_of(mid))) >= least) hi = mid; else lo = mid;
    }
    if (hi > border.key + 1 || (border.ties && static_cast<double>(w(value_of(border.key))) < least)) border = Border{hi - 1, 0};
  }

  // The draw: a segment of the row a wave, then the pieces of the segment that has it, then its values.  Ties count in order.
  constexpr int E = Row<T>::E;
  const int64_t segment = (a.v + kWaves * E - 1) / (kWaves * E) * E;
  uint64_t sum = 0;
  uint32_t ties = 0;
  for (int64_t at = wave * segment + lane * E; at < min((wave + 1) * segment, static_cast<int64_t>(a.v)); at += 64 * E)
    row.piece(at, [&](float x, int) { sum += weight(x, ties); });
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    sum += __shfl_xor(static_cast<unsigned long long>(sum), off, 64);
    ties += __shfl_xor(ties, off, 64);
  }
  __syncthreads();
  if (lane == 0) {
    s.wave64[wave] = sum;
    s.wave32[wave] = ties;
  }
  __syncthreads();
  const uint64_t each = border.ties ? w(value_of(border.key)) : 0;
  uint64_t total = 0;
  uint32_t tied = 0;
  for (int i = 0; i < kWaves; ++i) {
    const uint32_t kept = min(s.wave32[i], border.ties - tied);
    tied += kept;
    total += s.wave64[i] + kept * each;
  }
  const double part = static_cast<double>(u < 0x1p-40f ? 0.f : fminf(u, 0x1.fffffep-1f)) * static_cast<double>(total);
  const uint64_t target = min(static_cast<uint64_t>(fmax(part, 0.0)), total - 1);       // the first whose sum is above it
  uint64_t done = 0;
  tied = 0;
  int seg = 0;
  for (;; ++seg) {
    const uint32_t kept = min(s.wave32[seg], border.ties - tied);
    const uint64_t next = done + s.wave64[seg] + kept * each;
    if (next > target || seg == kWaves - 1) break;
    done = next;
    tied += kept;
  }
  // the segment: a run of neighbouring values each thread
  const int64_t run = (segment + kThreads - 1) / kThreads, from = seg * segment + tid * run;
  const int64_t to = min(min(from + run, (seg + 1) * segment), static_cast<int64_t>(a.v));
  sum = 0;
  ties = 0;
  for (int64_t i = from; i < to; ++i) sum += weight(to_f32(row.x[i]), ties);
  uint64_t all, tiesbefore = before64(ties, s, all);
  const uint32_t had = min(static_cast<uint64_t>(border.ties), tied + tiesbefore);
  const uint32_t mine = min(static_cast<uint64_t>(border.ties), tied + tiesbefore + ties) - had;
  uint64_t start = done + before64(sum + mine * each, s, all);
  if (start <= target && start + sum + mine * each > target) {
    uint32_t seen = had;
    for (int64_t i = from; i < to; ++i) {
      uint32_t tie = 0;
      uint64_t wi = weight(to_f32(row.x[i]), tie);
      if (tie && seen < border.ties) {
        wi = each;
        ++seen;
      }
      start += wi;
      if (start > target) {
        a.tokens[blockIdx.x] = i;
        break;
      }
    }
  }
}

int32_t check(const wc_sample_args& p, const char* what) {
  WC_REQUIRE(dtype_size(p.dtype), WC_ERR_DTYPE, "%s: dtype %d", what, p.dtype);
  WC_REQUIRE(p.n >= 0 && p.m >= 0 && p.v >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(p.v < (1ll << 30) && mul_sat({p.n, p.m}) < (1ll << 22), WC_ERR_LIMIT, "%s: 2^30 logits of a row or 2^22 rows, or more", what);
  return WC_OK;
}

}  // namespace
}  // namespace wc

extern "C" int64_t wc_sample_workspace_bytes(const wc_sample_args* args) {
  using namespace wc;
  clear_error();
  if (!args) {
    set_error(WC_ERR_NULL, "wc_sample: null args");
    return -1;
  }
  return check(*args, "wc_sample") ? -1 : 0;
}

extern "C" int32_t wc_sample(const wc_sample_args* args, void* stream) {
  using namespace wc;
  clear_error();
  const char* what = "wc_sample";
  WC_REQUIRE(args, WC_ERR_NULL, "%s: null args", what);
  const wc_sample_args& p = *args;
  if (int32_t rc = check(p, what)) return rc;
  if (p.n == 0 || p.m == 0) return WC_OK;
  const int es = dtype_size(p.dtype);
  WC_REQUIRE(p.v > 0, WC_ERR_SHAPE, "%s: rows without logits", what);
  WC_REQUIRE(p.logits && p.u && p.temperature && p.top_k && p.top_p && p.min_p && p.tokens, WC_ERR_NULL, "%s: null pointer", what);
  WC_REQUIRE(p.x_rows_inner > 0, WC_ERR_ARG, "%s: rows_inner must be positive", what);
  WC_REQUIRE(p.x_rows_inner < (1ll << 31), WC_ERR_LIMIT, "%s: rows_inner beyond 32 bits", what);
  WC_REQUIRE(aligned(p.logits, es) && aligned(p.u, 4) && aligned(p.temperature, 4) && aligned(p.top_k, 4) && aligned(p.top_p, 4) &&
                 aligned(p.min_p, 4) && aligned(p.tokens, 8),
             WC_ERR_ALIGN, "%s: pointers must be aligned to their elements", what);
  Sample a;
  a.x = static_cast<const char*>(p.logits);
  a.u = p.u;
  a.temperature = p.temperature;
  a.top_p = p.top_p;
  a.min_p = p.min_p;
  a.top_k = p.top_k;
  a.tokens = p.tokens;
  a.xn = p.x_stride_n;
  a.xo = p.x_stride_outer;
  a.xi = p.x_stride_inner;
  a.tn = p.temperature_stride_n;
  a.tm = p.temperature_stride_m;
  a.kn = p.top_k_stride_n;
  a.km = p.top_k_stride_m;
  a.pn = p.top_p_stride_n;
  a.pm = p.top_p_stride_m;
  a.mn = p.min_p_stride_n;
  a.mm = p.min_p_stride_m;
  a.v = static_cast<int32_t>(p.v);
  int bits = 0;
  while ((1ll << bits) < p.v) ++bits;
  a.fraction = std::min(48, 63 - bits);
  a.by_m = make_fastdiv(static_cast<uint32_t>(p.m));
  a.by_rows = make_fastdiv(static_cast<uint32_t>(p.x_rows_inner));
  const uint32_t rows = static_cast<uint32_t>(p.n * p.m);
  const hipStream_t s = as_stream(stream);
  if (p.dtype == WC_F32)
    sample_kernel<float><<<rows, kThreads, 0, s>>>(a);
  else if (p.dtype == WC_BF16)
    sample_kernel<bf16><<<rows, kThreads, 0, s>>>(a);
  else
    sample_kernel<f16><<<rows, kThreads, 0, s>>>(a);
  return check_launch(what);
}
