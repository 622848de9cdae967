// Draws a token of every row of logits by temperature, top-k, top-p and min-p, from a given random number.
//
//   w_i = exp((x_i - max x) / t);  kept: the first of the order (value down, index up);  the token is the lowest kept
//   index up to which the kept weights pass u times their sum
//
// The filters all keep the first of one order, so a kept set is a cut: a value, all above it, and those equal to it up to an
// index.  A row of logits is cut into chunks.  The first kernel has a workgroup for each chunk, which brings it into
// registers, finds its largest value, sums its weights and, where something is filtered, counts and sums them in bins: an
// eighth of a power of two of the weight each, so a bin holds a small part of the values and what lies above it is known without
// looking again.  The second has a workgroup for each row: it adds the chunks' bins up, finds the bin in which the cut falls,
// gathers what the bin holds (or all that may be kept, where that is little), finds the cut there, then the chunk that
// holds the token by the sums, and the token in the chunk.
//
// A bin may hold more than a list: of rows as vocabularies' heads give them, of 131072 logits and more at a temperature of 1, the bin of
// top_p = 0.95 does (4400 values of 262144).  For top-p such a bin is parted by its values' bits in one more look at the row, and
// what is above the part with the cut goes to the chunks' sums; for min-p, whose least value is known, all that is kept does
// (128 rows of 200003 in bf16, top_p = 0.95: at a temperature of 0.7, where the bin fits, 89 us; of 1.0 134, over the digits of the
// whole row 1276).  What is left is cut on the values' bits, digit by digit, over the whole row: thousands of equal values at the cut, a
// top_k whose bin does not fit, and rows of one chunk, which are short (64 of 8000 with all values in a few bins: 33 us, spread 29).
//
// Which token comes out must not hang on the order of a sum, so weights are summed as whole numbers, of 2^-48 of the
// largest weight (more where rows are so long that 64 bits could not hold the sum): each is the exponential in 64 bits,
// off by 2^-46 of itself, and rounded once, to 1 at least, so that u = 0 gives the first that has a weight at all.  A chunk's are of its
// own largest, and its sums are brought to the row's units by a shift, to 1 at least.
//
// Those exponentials, some 20 operations in 64 bits a value and as many others, bound the first kernel by instructions: 256 rows of 131072 in fp32, unfiltered, 39 us
// (3.4 TB/s); with bins, an atomic in LDS a value more, 128 of 100003 in bf16 25 us (5.2e11 values a second; 8.6e11 without bins).
#include <algorithm>

#include "wc_answer_abi.h"
#include "wc_common.h"

namespace wc {
namespace {

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kDigitBits = 10, kDigits = 1 << kDigitBits;
static_assert(kDigits == 2 * kThreads, "two digits a thread");
constexpr int kBinBits = 9, kBins = 1 << kBinBits;     // of an eighth of a power of two: weights down to 2^-64 of a chunk's largest
constexpr int kList = 2048;          // values that a row's workgroup sorts
constexpr int kRank = 128;           // values that are put in order by comparing each with each
constexpr int kChunkThreads = 512, kChunks = 64;     // chunks of a row at most

struct Sample {
  const char* x;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int64_t* tokens;
  int64_t xn, xo, xi, tn, tm, kn, km, pn, pm, mn, mm;
  int32_t v, fraction;       // fraction: bits below the largest weight that sums hold
  int32_t chunk, chunks;     // values of a chunk, chunks of a row
  struct ChunkSums* sums;    // [rows][chunks]
  FastDiv by_m, by_rows, by_chunks, by_chunk;
};

template <typename T>
__device__ __forceinline__ T larger(T a, T b) { return a > b ? a : b; }
template <typename T>
__device__ __forceinline__ T smaller(T a, T b) { return a < b ? a : b; }

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

// 2^(i / 64)
struct Powers {
  double v[64];
};
constexpr Powers powers() {
  Powers p = {};
  for (int i = 0; i < 64; ++i) {
    double term = 1, sum = 1;
    for (int k = 1; k < 20; ++k) sum += term *= 0.69314718055994530942 / 64 * i / k;
    p.v[i] = sum;
  }
  return p;
}
__constant__ const Powers kPowers = powers();

// Weights as whole numbers: 2^(y + fraction), y = x log2(e) / t - floor, with 2^(i/64) from a table and the rest, at most
// 2^-7 of a power, from the first terms of its series, whose next is under 2^-54.  `floor` is a whole number next to the
// largest value's x log2(e) / t, by which sums of different ones can be brought together; y is at most 2^-12, whatever t is,
// because it is counted from the largest value down.
constexpr uint64_t kMagic = 0x4330000000000000;      // 2^52 as a float of 64 bits: its last bits are a whole number added to it
struct Weights {
  const double* table;       // 64
  double scale, floor, at_top, most;
  float top;                 // the largest value; where it is infinite, only what is it has a weight
  int fraction;
  __device__ __forceinline__ Weights(const double* table, float top, float t, int fraction)
      : table(table), scale(1.4426950408889634074 / t), floor(0), at_top(0), most(top), top(top), fraction(fraction) {
    if (!(fabsf(top) < INFINITY)) return;
    const double p = most * scale;
    const bool fine = fabs(p) < 0x1p40;               // where a whole number is near enough
    floor = fine ? ceil(p) : p;
    at_top = fine ? fma(most, scale, -floor) : 0.0;
  }
  // The weight and kMagic, where the largest value is finite; NaN and -infinity have none.  The series' terms are in registers
  // (`c`, of terms()): a constant would be brought into one for every fused multiply-add.
  struct Terms {
    double c[6];
  };
  static __device__ __forceinline__ Terms terms() {
    constexpr double l = 0.69314718055994530942 / 64;
    Terms t = {{1.0, l, l * l / 2, l * l * l / 6, l * l * l * l / 24, l * l * l * l * l / 120}};
#pragma unroll
    for (int i = 0; i < 6; ++i) asm volatile("" : "+v"(t.c[i]));
    return t;
  }
  __device__ __forceinline__ uint64_t finite_and_magic(float x, const Terms& t) const {
    double y = fma(static_cast<double>(x) - most, scale, at_top);
    const double some = y > -1075.0 ? 1.0 : 0.0;     // 0 under what 64 bits hold
    asm("v_max_f64 %0, %1, %2" : "=v"(y) : "v"(y), "v"(-200.0));       // far under a unit, and the exponent below stays one; -200 of NaN
    constexpr double magic = 0x1.8p52;
    const double n = fma(y, 64.0, magic);
    const int i = static_cast<int>(static_cast<uint32_t>(__builtin_bit_cast(uint64_t, n)));
    const double f = fma(y, 64.0, magic - n);
    double p = fma(t.c[5], f, t.c[4]);
    p = fma(p, f, t.c[3]);
    p = fma(p, f, t.c[2]);
    p = fma(p, f, t.c[1]);
    p = fma(p, f, t.c[0]);
    // times 2^(i / 64 + fraction), whole powers as its exponent
    const uint64_t bits = __builtin_bit_cast(uint64_t, p * table[i & 63]);
    const uint32_t high = static_cast<uint32_t>(bits >> 32) + (static_cast<uint32_t>(i & ~63) << 14) + (static_cast<uint32_t>(fraction) << 20);
    p = __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(bits));
    asm("v_max_f64 %0, %1, %2" : "=v"(p) : "v"(p), "v"(some));
    return __builtin_bit_cast(uint64_t, p + 0x1p52);
  }
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (top == INFINITY) return x == top ? 1ull << fraction : 0;
    return finite_and_magic(x, terms()) - kMagic;
  }
};

// What the first kernel leaves of a chunk
struct ChunkSums {
  uint64_t weight[kBins];    // of each bin, for rows with a filter, as far as Rules::bins() asks for them
  uint32_t count[kBins];
  double floor;              // of its weights
  uint64_t sum;
  uint32_t top, first;       // key of the largest value and its index
};

// The filters of a row
struct Rules {
  float t, top_p, min_p;
  int32_t top_k;
  __device__ __forceinline__ Rules(const Sample& a, uint32_t model, uint32_t r)
      : t(a.temperature[model * a.tn + r * a.tm]), top_p(a.top_p[model * a.pn + r * a.pm]),
        min_p(a.min_p[model * a.mn + r * a.mm]), top_k(a.top_k[model * a.kn + r * a.km]) {}
  __device__ __forceinline__ bool greedy() const { return !(t > 0.f) || top_k == 1 || top_p <= 0.f; }
  __device__ __forceinline__ bool filter(int v) const { return (top_k > 0 && top_k < v) || top_p < 1.f || min_p > 0.f; }
  // What is wanted of the bins, each an atomic for every value: of a top_k whose values fit a list, where the rest is found,
  // the counts; of a longer one both; else the weights, which say how many there can be.
  __device__ __forceinline__ bool counts(int v) const { return top_k > 0 && top_k < v; }
  __device__ __forceinline__ bool weights(int v) const { return !(counts(v) && top_k <= kList / 2); }
};

// Bins: floor(8 x log2(e) / t) counted down from that of the largest value
struct Bins {
  float scale, base;
  __device__ __forceinline__ Bins(float t, float top) : scale(fmaxf(8 * 1.44269504f / t, 1e-45f)) { base = place(top); }
  __device__ __forceinline__ float scaled(float x) const { return fminf(fmaxf(x * scale, -1e30f), 1e30f); }
  __device__ __forceinline__ float place(float x) const { return floorf(scaled(x)); }
  __device__ __forceinline__ int operator()(float x) const { return static_cast<int>(fminf(base - place(x), kBins - 1)); }
};

// The border of a kept set: all keys above `key`, and the first `ties` of those that are it.
struct Border {
  uint32_t key;
  uint32_t ties;
};

struct Shared {
  union {
    struct {
      uint64_t weight[kDigits];
      uint32_t count[kDigits];
    };
    struct {
      uint64_t list[kList], other[kList];                  // key, then what is left of all ones by the index: ordered as values are
      uint64_t bin_weight[kBins], above_weight[kBins];     // of a bin, of all before it
      uint32_t bin_count[kBins], above_count[kBins];
      uint64_t rank_weight[kRank], rank_before[kRank];
      uint32_t rank[kRank];
      uint64_t chunk_sum[kChunks];
    };
  };
  double table[64];
  uint64_t wave64[kWaves], ends[kWaves][2];
  uint32_t wave32[kWaves];
  uint64_t found64[2];
  uint32_t found32[4];
};

// value e of a vector
template <typename T>
__device__ __forceinline__ float value_in(const u32x4& v, int e) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(float, static_cast<uint32_t>(v[e]));
  } else if constexpr (std::is_same<T, bf16>::value) {
    return e & 1 ? bf16_hi(v[e / 2]) : bf16_lo(v[e / 2]);
  } else {
    return static_cast<float>(__builtin_bit_cast(f16, static_cast<uint16_t>(v[e / 2] >> (e & 1) * 16)));
  }
}

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
  // A thread's values eight pieces at a time, all on their way together: go(piece, its first value's index, how many of its values
  // were in the piece before).
  template <typename F>
  __device__ __forceinline__ void batches(F go) const {
    constexpr int step = kThreads * E;
    for (int64_t at = static_cast<int64_t>(threadIdx.x) * E; at < v; at += 8 * step) {
      u32x4 t[8];
      int64_t from[8];
      int skip[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // a piece over the end from further left, where what is not its own is left out
        const int64_t own = at + i * step;
        from[i] = v >= E ? smaller(own, static_cast<int64_t>(v - E)) : 0;
        skip[i] = static_cast<int>(smaller(own - from[i], static_cast<int64_t>(E)));
        if (v >= E) {
          __builtin_memcpy(&t[i], x + from[i], 16);
        } else {
          T few[E];
#pragma unroll
          for (int e = 0; e < E; ++e) few[e] = x[e < v ? e : 0];
          __builtin_memcpy(&t[i], few, 16);
        }
      }
      go(t, from, skip);
    }
  }
  template <typename F>
  __device__ __forceinline__ void all(F go) const {
    batches([&](const u32x4(&t)[8], const int64_t(&from)[8], const int(&skip)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (e >= skip[i] && e < v) go(value_in<T>(t[i], e), static_cast<int>(from[i]) + e);
    });
  }
  // put(index, place) of the values within [lo, hi], places from take(how many a wave has): a bit for each of a thread's 8 E values
  // at a time, while the next are on their way (AHEAD), then a turn for each bit.
  template <bool AHEAD, typename G, typename F>
  __device__ __forceinline__ void select(float lo, float hi, G take, F put) const {
    constexpr int step = kThreads * E;
    if (v < E) {
      const float f = static_cast<int>(threadIdx.x) < v ? to_f32(x[threadIdx.x]) : __builtin_nanf("");
      if (f >= lo && f <= hi) put(threadIdx.x, take(1));
      return;
    }
    const uint32_t last = v - E;                       // pieces over the end from there, where what is not their own is left out
    auto load = [&](uint32_t at, u32x4(&t)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) __builtin_memcpy(&t[i], x + smaller(at + i * step, last), 16);
    };
    const int lane = threadIdx.x & 63;
    const uint32_t end = v, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 64 * E;
    u32x4 t[8], next[8];
    uint32_t first = wave;                             // of the wave: the same for its lanes
    if (AHEAD && first < end) load(first + lane * E, t);
    for (; first < end; first += 8 * step) {
      const uint32_t at = first + lane * E;
      if (!AHEAD) load(at, t);
      if (AHEAD && first + 8 * step < end) load(at + 8 * step, next);
      uint64_t mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float f = value_in<T>(t[i], e);
          m |= __builtin_amdgcn_fmed3f(f, lo, hi) == f ? 1u << e : 0u;
        }
        mine |= static_cast<uint64_t>(m) << i * E;
      }
      if (first + 7 * step + 64 * E > end) {           // the wave's last: pieces that begin before their own place, or have none
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t own = at + i * step;
          const uint32_t skip = smaller(own - smaller(own, last), static_cast<uint32_t>(E));
          const uint64_t bits = ~0u << skip & ((1u << E) - 1);
          mine &= bits << i * E | ~(((1ull << E) - 1) << i * E);
        }
      }
      if (__ballot(mine != 0)) {
        const int n = __popcll(mine);
        int upto = n;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const int up = __shfl_up(upto, off, 64);
          if (lane >= off) upto += up;
        }
        int place = 0;
        if (lane == 63) place = take(upto);
        place = __builtin_amdgcn_readlane(place, 63) + upto - n;
        while (mine) {
          const int bit = __ffsll(static_cast<unsigned long long>(mine)) - 1;
          mine &= mine - 1;
          put(static_cast<int>(smaller(at + bit / E * step, last)) + bit % E, place++);
        }
      }
#pragma unroll
      for (int i = 0; AHEAD && i < 8; ++i) t[i] = next[i];
    }
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
  // every lane of 16 has a wave's sum
  uint64_t mine = s.wave64[lane & (kWaves - 1)], upto = mine;
#pragma unroll
  for (int off = 1; off < kWaves; off <<= 1) {
    const uint64_t up = __shfl_up(static_cast<unsigned long long>(upto), off, kWaves);
    if ((lane & (kWaves - 1)) >= off) upto += up;
  }
  total = __shfl(static_cast<unsigned long long>(upto), kWaves - 1, 64);
  return __shfl(static_cast<unsigned long long>(upto - mine), wave, 64) + sum - v;
}

// the sum over the workgroup
__device__ __forceinline__ uint64_t sum64(uint64_t v, Shared& s) {
#pragma unroll
  for (int off = 32; off; off >>= 1) v += __shfl_xor(static_cast<unsigned long long>(v), off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave64[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s.wave64[threadIdx.x & (kWaves - 1)];
#pragma unroll
  for (int off = kWaves / 2; off; off >>= 1) v += __shfl_xor(static_cast<unsigned long long>(v), off, 64);
  return v;
}

// The border at which what is kept from the top first reaches `limit`, of counts (COUNT) or of weights; limit > 0 and at
// most what all keys above kNever have.  Keys above `from` count, and the first `ties` of those that are it.
template <bool COUNT, typename T>
__device__ Border find_border(const Row<T>& row, const Weights& w, Shared& s, uint32_t top, Border from, uint64_t limit) {
  uint32_t lo = larger(from.key, kNever + 1), hi = top;
  uint64_t above = 0;
  for (;;) {
    const uint32_t width = hi - lo;
    const int shift = larger(0, 32 - __clz(width | 1) - kDigitBits);          // digits of 2^shift keys, at most kDigits
    __syncthreads();
    for (int i = threadIdx.x; i < kDigits; i += kThreads) {
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
    const int b1 = kDigits - 1 - 2 * threadIdx.x, b0 = b1 - 1;
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
      return Border{lo, static_cast<uint32_t>(smaller((left + each - 1) / each, have))};
    }
    hi = smaller(hi, lo + ((1u << shift) - 1));
  }
}

// the unit that the number u falls on
__device__ __forceinline__ uint64_t pick(float u, uint64_t total) {
  const double part = static_cast<double>(u < 0x1p-40f ? 0.f : fminf(u, 0x1.fffffep-1f)) * static_cast<double>(total);
  return smaller(static_cast<uint64_t>(fmax(part, 0.0)), total - 1);               // the first whose sum is above it
}

// The least key that min_p keeps, of which `power` is the logarithm: by the value's distance from the largest one, because the whole
// number that is its weight is rounded, and 1 for all that are small enough.  Lanes try 64 keys at a time: neighbours, then some
// of all there are.
__device__ __forceinline__ uint32_t least_key(const Weights& w, uint32_t top, double power) {
  if (w.top == INFINITY) return top;
  const int lane = threadIdx.x & 63;
  uint32_t lo = kNever, hi = top;                    // hi is kept, lo not
  auto keeps = [&](uint32_t key) __attribute__((always_inline)) { return (static_cast<double>(value_of(key)) - w.most) * w.scale >= power; };
  // next to where it must be, as a rule (a row of 32000 with every filter: 17.3 us, by the search alone 18.1)
  const uint32_t near = key_of(static_cast<float>(fmax(w.most + power / w.scale, -3.4e38))) - 32;
  int first = __ffsll(static_cast<unsigned long long>(__ballot(near + lane >= hi || keeps(near + lane)))) - 1;
  if (first > 0) return smaller(near + first, hi);
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
    first = __ffsll(static_cast<unsigned long long>(__ballot(at >= hi || keeps(at)))) - 1;
    lo += first * step;
    hi = smaller(hi, lo + step);
  }
  return hi;
}

// Of the values with keys [klo, khi], which are more than a list holds, those next to the place where weights summed from the top
// and from `above` on reach the limit: into s.list, the sum above them into s.found64[0] and the weights between them and khi that
// min_p keeps into s.chunk_sum, by their chunks.  How many are listed, or -1 where more than a list holds are equal.
template <typename T>
__device__ __forceinline__ int part_bin(Row<T> row, Weights w, Shared& s, uint32_t klo, uint32_t khi, uint32_t least, uint64_t above, uint64_t limit,
                                        FastDiv by_chunk) {
  const int tid = threadIdx.x;
  const auto none = [](int) { return 0; };
  uint32_t lo = klo, hi = khi;
  for (;;) {
    const uint32_t width = hi - lo;
    const int shift = larger(0, 32 - __clz(width | 1) - kDigitBits);          // parts of 2^shift keys, at most kDigits
    __syncthreads();
    for (int i = tid; i < kDigits; i += kThreads) {
      s.weight[i] = 0;
      s.count[i] = 0;
    }
    if (tid == 0) s.found32[0] = 0, s.found64[0] = above;
    __syncthreads();
    row.template select<false>(value_of(lo), value_of(hi), none, [&](int i, int) {
      const float x = to_f32(row.x[i]);
      const uint32_t k = key_of(x);
      if (k < lo || k > hi) return;                    // a zero of the other sign
      atomicAdd(&s.count[(k - lo) >> shift], 1u);
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.weight[(k - lo) >> shift]), static_cast<unsigned long long>(w(x)));
    });
    __syncthreads();
    // parts from the top, two a thread: the first that reaches the limit; where rounding leaves that behind all, the last that has any
    const int d1 = kDigits - 1 - 2 * tid, d0 = d1 - 1;
    const uint64_t v1 = s.weight[d1], v0 = s.weight[d0];
    uint64_t total;
    const uint64_t had1 = above + before64(v1 + v0, s, total), had0 = had1 + v1;
    if (v1 && had1 < limit && (had0 >= limit || had0 == above + total)) s.found32[0] = d1, s.found64[0] = had1;
    if (v0 && had0 < limit && (had0 + v0 >= limit || had0 + v0 == above + total)) s.found32[0] = d0, s.found64[0] = had0;
    __syncthreads();
    const uint32_t part = s.found32[0], n = s.count[part];
    above = s.found64[0];
    lo += part << shift;
    hi = smaller(hi, lo + ((1u << shift) - 1));
    if (n <= kList) break;
    if (shift == 0) return -1;
  }
  __syncthreads();
  if (tid == 0) s.found32[1] = 0;
  if (tid < kChunks) s.chunk_sum[tid] = 0;
  __syncthreads();
  row.template select<false>(value_of(lo), value_of(khi), none, [&](int i, int) {
    const float x = to_f32(row.x[i]);
    const uint32_t k = key_of(x);
    if (k < lo || k > khi) return;
    if (k <= hi)
      s.list[atomicAdd(&s.found32[1], 1u)] = static_cast<uint64_t>(k) << 32 | ~static_cast<uint32_t>(i);
    else if (k >= least)
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.chunk_sum[fdiv(static_cast<uint32_t>(i), by_chunk)]), static_cast<unsigned long long>(w(x)));
  });
  __syncthreads();
  return static_cast<int>(s.found32[1]);
}

// The draw by the digits of keys, over the whole row.
template <typename T>
__device__ __attribute__((noinline)) void draw_by_digits(Row<T> row, Weights w, Shared& s, Rules rules, uint32_t top, uint32_t least, float u,
                                                         int64_t* token) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float top_p = rules.top_p;
  const int32_t top_k = rules.top_k;
  Border border{kNever, 0};
  if (top_k > 0 && top_k < row.v) {
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
    const uint64_t limit = larger(static_cast<uint64_t>(ceil(part)), static_cast<uint64_t>(1));
    border = find_border<false>(row, w, s, top, border, smaller(limit, total));
  }
  if (least > border.key) border = Border{least - 1, 0};

  // The draw: a segment of the row a wave, then the pieces of the segment that has it, then its values.  Ties count in order.
  constexpr int E = Row<T>::E;
  const int64_t segment = (row.v + kWaves * E - 1) / (kWaves * E) * E;
  uint64_t sum = 0;
  uint32_t ties = 0;
  for (int64_t at = wave * segment + lane * E; at < smaller((wave + 1) * segment, static_cast<int64_t>(row.v)); at += 64 * E)
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
    const uint32_t kept = smaller(s.wave32[i], border.ties - tied);
    tied += kept;
    total += s.wave64[i] + kept * each;
  }
  const uint64_t target = pick(u, total);
  uint64_t done = 0;
  tied = 0;
  int seg = 0;
  for (;; ++seg) {
    const uint32_t kept = smaller(s.wave32[seg], border.ties - tied);
    const uint64_t next = done + s.wave64[seg] + kept * each;
    if (next > target || seg == kWaves - 1) break;
    done = next;
    tied += kept;
  }
  // the segment: a run of neighbouring values each thread
  const int64_t run = (segment + kThreads - 1) / kThreads, from = seg * segment + tid * run;
  const int64_t to = smaller(smaller(from + run, (seg + 1) * segment), static_cast<int64_t>(row.v));
  sum = 0;
  ties = 0;
  for (int64_t i = from; i < to; ++i) sum += weight(to_f32(row.x[i]), ties);
  uint64_t all, tiesbefore = before64(ties, s, all);
  const uint32_t had = smaller(static_cast<uint64_t>(border.ties), tied + tiesbefore);
  const uint32_t mine = smaller(static_cast<uint64_t>(border.ties), tied + tiesbefore + ties) - had;
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
        *token = i;
        break;
      }
    }
  }
}


// A workgroup's chunk of a row: its largest value, the sum of its weights, and its bins.
struct ChunkShared {
  uint64_t weight[kBins], red[kChunkThreads / 64];
  uint32_t count[kBins];
  double table[64];
  float tops[kChunkThreads / 64];
};
template <typename T>
__device__ __forceinline__ void sum_chunk(const Sample& a, ChunkShared& s, ChunkSums& out) {
  constexpr int E = Row<T>::E, NW = kChunkThreads / 64, KEPT = 16 / E;       // 16 values a thread stay in registers
  uint64_t *const weight = s.weight, *const red = s.red;
  uint32_t* const count = s.count;
  double* const table = s.table;
  float* const tops = s.tops;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t rowi = fdiv(blockIdx.x, a.by_chunks), c = blockIdx.x - rowi * a.by_chunks.d;
  const uint32_t model = fdiv(rowi, a.by_m), r = rowi - model * a.by_m.d, outer = fdiv(r, a.by_rows);
  const int64_t lo = static_cast<int64_t>(c) * a.chunk;
  const int n = static_cast<int>(smaller(static_cast<int64_t>(a.chunk), a.v - lo));
  const T* x = reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (r - outer * a.by_rows.d) * a.xi + lo;
  auto load = [&](int at, T(&v)[E]) {
    if (at + E <= n) {
      __builtin_memcpy(v, x + at, 16);               // at element alignment
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = at + e < n ? x[at + e] : from_f32<T>(-INFINITY);
    }
  };
  T kept[KEPT][E];
#pragma unroll
  for (int i = 0; i < KEPT; ++i) load((i * kChunkThreads + tid) * E, kept[i]);
  const Rules rules(a, model, r);
  if (tid < 64) table[tid] = kPowers.v[tid];
  for (int i = tid; i < kBins; i += kChunkThreads) weight[i] = 0, count[i] = 0;
  float top = -INFINITY;
  auto look = [&](const T(&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) top = fmaxf(top, to_f32(v[e]));       // takes no notice of NaN
  };
#pragma unroll
  for (int i = 0; i < KEPT; ++i) look(kept[i]);
  for (int at = (KEPT * kChunkThreads + tid) * E; at < n; at += kChunkThreads * E) {
    T v[E];
    load(at, v);
    look(v);
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if (lane == 0) tops[wave] = top;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < NW; ++v) top = fmaxf(top, tops[v]);
  const Weights w(table, top, rules.t, a.fraction);
  if (tid == 0) {
    out.top = key_of(top);
    out.floor = w.floor;
    out.first = static_cast<uint32_t>(lo);
    out.sum = 0;
  }
  if (top == -INFINITY) return;
  if (rules.greedy()) {
    // the lowest index with the largest value
    uint32_t first = 0xffffffffu;
    auto find = [&](const T(&v)[E], int at) {
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (to_f32(v[e]) == top) first = smaller(first, static_cast<uint32_t>(at + e));
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i) find(kept[i], (i * kChunkThreads + tid) * E);
    for (int at = (KEPT * kChunkThreads + tid) * E; at < n; at += kChunkThreads * E) {
      T v[E];
      load(at, v);
      find(v, at);
    }
#pragma unroll
    for (int off = 32; off; off >>= 1) first = smaller(first, static_cast<uint32_t>(__shfl_xor(static_cast<int>(first), off, 64)));
    if (lane == 0) red[wave] = first;
    __syncthreads();
    if (tid == 0) {
      for (int v = 1; v < NW; ++v) first = smaller(first, static_cast<uint32_t>(red[v]));
      out.first = static_cast<uint32_t>(lo) + first;
    }
    return;
  }
  const bool filter = rules.filter(a.v), counts = rules.counts(a.v), weights = rules.weights(a.v);
  const Bins bins(rules.t, top);
  uint64_t sum = 0;                                  // of weights and kMagic each: 64 bits wrap, and what is right comes back
  int added = 0;
  const Weights::Terms terms = Weights::terms();
  auto add = [&](const T(&v)[E]) __attribute__((always_inline)) {
    if (top == INFINITY) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = to_f32(v[e]);
        if (filter && f > -INFINITY) {
          if (counts) atomicAdd(&count[bins(f)], 1u);
          if (weights) atomicAdd(reinterpret_cast<unsigned long long*>(&weight[bins(f)]), static_cast<unsigned long long>(w(f)));
        } else if (!filter) {
          sum += w(f);
        }
      }
    } else if (!filter) {
#pragma unroll
      for (int e = 0; e < E; ++e) sum += w.finite_and_magic(to_f32(v[e]), terms);
      added += E;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float f = to_f32(v[e]);
        if (f > -INFINITY) {
          const int b = bins(f);
          if (counts) atomicAdd(&count[b], 1u);
          if (weights) atomicAdd(reinterpret_cast<unsigned long long*>(&weight[b]), static_cast<unsigned long long>(w.finite_and_magic(f, terms) - kMagic));
        }
      }
    }
  };
#pragma unroll
  for (int i = 0; i < KEPT; ++i) add(kept[i]);
  for (int at = (KEPT * kChunkThreads + tid) * E; at < n; at += kChunkThreads * E) {
    T v[E];
    load(at, v);
    add(v);
  }
  if (filter) {
    __syncthreads();
    for (int i = tid; i < kBins; i += kChunkThreads) {
      if (weights) out.weight[i] = weight[i], sum += weight[i];
      if (counts) out.count[i] = count[i];
    }
  }
  sum -= added * kMagic;
#pragma unroll
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(static_cast<unsigned long long>(sum), off, 64);
  if (lane == 0) red[wave] = sum;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int v = 1; v < NW; ++v) sum += red[v];
    out.sum = sum;
  }
}
template <typename T>
__global__ __launch_bounds__(kChunkThreads) void sample_chunks_kernel(Sample a) {
  __shared__ ChunkShared s;
  sum_chunk<T>(a, s, a.sums[blockIdx.x]);
}

// The rank of each of n <= kRank different values among them, from the largest down, and the sum of the weights (in
// rank_weight) of those before it.  A wave compares 64 of them with its share of all.
__device__ void rank_all(const uint64_t* list, int n, Shared& s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kRank; i += kThreads) s.rank[i] = 0, s.rank_before[i] = 0;
  __syncthreads();
  constexpr int kParts = kWaves * 64 / kRank;
  const int i = wave / kParts * 64 + lane;
  const uint64_t v = i < n ? list[i] : 0;
  uint32_t rank = 0;
  uint64_t sum = 0;
  for (int j = wave % kParts; j < n; j += kParts) {
    const bool before = list[j] > v;
    rank += before;
    sum += before ? s.rank_weight[j] : 0;
  }
  if (i < n) {
    atomicAdd(&s.rank[i], rank);
    atomicAdd(reinterpret_cast<unsigned long long*>(&s.rank_before[i]), static_cast<unsigned long long>(sum));
  }
  __syncthreads();
}

// A row's token.  WHOLE: rows are one chunk each, and their workgroups sum it first, which saves a launch (128 greedy rows of 1000: 6.1
// and 4.9 us), with registers for two workgroups a unit instead of one, at the price of some in scratch memory (fp32 7, fp16 16, bf16
// 75 of them: 518 rows of 185 in bf16 by top-k and top-p 33.6 us, by one workgroup 40.5; 58 of 829 by top-p and min-p 16.5 and 14.6).
// Latency bounds it: a row's bins, its list and its token are some 30 steps that wait for each other, 39 us for 128 rows of 100003 (25.6 MB,
// of which each row is read once more to fill the list).
template <typename T, bool WHOLE>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(WHOLE ? 4 : 2))) void sample_rows_kernel(Sample a) {
  static_assert(kThreads == kChunkThreads, "one workgroup does both");
  __shared__ Shared s;
  __shared__ ChunkSums whole;
  if constexpr (WHOLE) {
    __shared__ ChunkShared c;
    sum_chunk<T>(a, c, whole);
    __syncthreads();
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t model = fdiv(blockIdx.x, a.by_m), r = blockIdx.x - model * a.by_m.d, outer = fdiv(r, a.by_rows);
  const Row<T> row{reinterpret_cast<const T*>(a.x) + model * a.xn + outer * a.xo + (r - outer * a.by_rows.d) * a.xi, a.v};
  const ChunkSums* const chunks = [&]() __attribute__((always_inline)) -> const ChunkSums* {
    if constexpr (WHOLE) return &whole;
    else return a.sums + static_cast<int64_t>(blockIdx.x) * a.chunks;
  }();
  // every wave: lane c has chunk c
  const bool mine = lane < a.chunks;
  const ChunkSums& my = chunks[mine ? lane : 0];
  const uint32_t my_top = mine ? my.top : 0, my_first = mine ? my.first : 0xffffffffu;
  const double my_floor = my.floor;
  const uint64_t my_sum = mine ? my.sum : 0;
  const Rules rules(a, model, r);
  const double power = rules.min_p > 0.f ? log2(static_cast<double>(fminf(rules.min_p, 1.f))) : 0.0;      // while the chunks' sums are on their way
  const float u = a.u[blockIdx.x];
  int64_t* const token = a.tokens + blockIdx.x;
  if (tid < 64) s.table[tid] = kPowers.v[tid];
  uint64_t best = static_cast<uint64_t>(my_top) << 32 | static_cast<uint32_t>(~my_first);
#pragma unroll
  for (int off = 32; off; off >>= 1) best = larger(best, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(best), off, 64)));
  const uint32_t top = best >> 32, first = ~static_cast<uint32_t>(best);
  if (top <= kNever || rules.greedy()) {
    if (tid == 0) *token = top <= kNever ? -1 : static_cast<int64_t>(first);
    return;
  }
  const Weights w(s.table, value_of(top), rules.t, a.fraction);
  const Bins bins(rules.t, w.top);
  // a chunk's sums in the row's units: right by so many bits, something stays something while 64 bits would hold it
  const double my_shift = w.top == INFINITY && my_top != top ? INFINITY : fmax(w.floor - my_floor, 0.0);
  const float my_off = my_top > kNever ? bins.base - bins.place(value_of(my_top)) : 0.f;
  auto units = [&](uint64_t v, double shift) __attribute__((always_inline)) {
    return v && shift < 1075 ? larger(shift < 64 ? v >> static_cast<int>(shift) : 0, static_cast<uint64_t>(1)) : 0;
  };

  // the kept: keys above cut_key, and those that are it up to index cut_last
  uint32_t cut_key = kNever, cut_last = 0;
  int list_from = kBins, listed = 0;             // all of the bins before list_from are kept, and what of the list is
  bool parted = false;                           // and what is above the list in its bin, in the chunks' sums already
  bool filter = rules.filter(a.v);
  // what min_p keeps: keys from `least` on, of weights of 2^power of the largest or more
  const uint32_t least = rules.min_p > 0.f ? least_key(w, top, power) : kNever + 1;
  __syncthreads();
  auto kept = [&](uint32_t k, uint32_t i) __attribute__((always_inline)) { return k >= least && (k > cut_key || (k == cut_key && i <= cut_last)); };
  auto list_key = [&](uint64_t v) { return static_cast<uint32_t>(v >> 32); };
  auto list_index = [&](uint64_t v) { return ~static_cast<uint32_t>(v); };
  if (filter) {
    // the row's bins and what is above each
    for (int i = tid; i < kBins; i += kThreads) s.bin_weight[i] = 0, s.bin_count[i] = 0;
    __syncthreads();
    // f(bin, the chunk's shift, i): of the values i of all chunks, a wave's of one chunk, eight a thread on their way
    auto add_bins = [&](const auto* first, auto f) __attribute__((always_inline)) {
      for (int i0 = tid; i0 < a.chunks * kBins; i0 += 8 * kThreads) {
        auto v = *first;
        decltype(v) all[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {               // past the last, the last again
          const int i = smaller(i0 + q * kThreads, a.chunks * kBins - 64 + lane);
          all[q] = *reinterpret_cast<decltype(first)>(reinterpret_cast<const char*>(first) + sizeof(ChunkSums) * (i / kBins) + sizeof(v) * (i % kBins));
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int i = i0 + q * kThreads, c = smaller(i / kBins, a.chunks - 1);
          const float off = __shfl(my_off, c, 64);
          const double shift = __shfl(my_shift, c, 64);
          // nothing has been written of a chunk without values
          if (__shfl(my_top, c, 64) > kNever && i < a.chunks * kBins && all[q])
            f(static_cast<int>(fminf(i % kBins + off, kBins - 1)), shift, all[q]);
        }
      }
    };
    const bool counts = rules.counts(a.v), weights = rules.weights(a.v);
    if (counts) add_bins(chunks->count, [&](int b, double, uint32_t n) { atomicAdd(&s.bin_count[b], n); });
    if (weights)
      add_bins(chunks->weight, [&](int b, double shift, uint64_t v) {
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.bin_weight[b]), static_cast<unsigned long long>(units(v, shift)));
      });
    __syncthreads();
    uint64_t total = 0, all = 0, aw = 0;
    const uint64_t bw = tid < kBins ? s.bin_weight[tid] : 0;
    // how many there are, or can be at most: a value of bin b has at least 2^(-(b + 1) / 8) of the largest
    // weight, which is at least half of all its bits
    uint32_t bc = 0;
    if (tid < kBins)
      bc = counts ? s.bin_count[tid] : static_cast<uint32_t>(fmin(1e6, ceil(static_cast<double>(bw) * exp2f((tid + 10) / 8.f) * ldexp(1.0, -a.fraction))));
    const uint64_t ac = before64(bc, s, all);
    if (weights) aw = before64(bw, s, total);
    if (tid < kBins) {
      s.above_weight[tid] = aw;
      s.above_count[tid] = ac;
      s.bin_count[tid] = bc;
    }
    __syncthreads();
    // the first bin with which a sum from the top reaches the limit; the last where none does
    auto find_bin = [&](const auto* above, uint64_t limit) __attribute__((always_inline)) {
      int lo = 0;
#pragma unroll
      for (int step = kBins / 2; step; step /= 2)
        if (lo + step < kBins && above[lo + step] < limit) lo += step;
      return lo;
    };
    // The values of bins [b0, b1], whose places are under the upper edge of b0 and from the lower edge of b1 on: places rise with values,
    // so the last and first of them are next to the edges divided by the scale.  A lane has a candidate.
    auto edges = [&](int b0, int b1, float& lo, float& hi) __attribute__((always_inline)) {
      hi = INFINITY;
      lo = -3.402823466e38f;
      if (b0) {
        const float edge = bins.base - b0 + 1, at = value_of(key_of(edge / bins.scale) + 16 - lane);
        hi = __shfl(at, (__ffsll(static_cast<unsigned long long>(__ballot(!(bins.scaled(at) >= edge)))) + 63) & 63, 64);
      }
      if (b1 < kBins - 1) {
        const float edge = bins.base - b1, at = value_of(key_of(edge / bins.scale) - 16 + lane);
        lo = __shfl(at, (__ffsll(static_cast<unsigned long long>(__ballot(!(bins.scaled(at) < edge)))) + 63) & 63, 64);
      }
    };
    // the values of bins [b0, b1] into the list; whether they fit
    auto gather = [&](int b0, int b1) __attribute__((always_inline)) {
      float lo, hi;
      edges(b0, b1, lo, hi);
      __syncthreads();
      if (tid == 0) s.found32[1] = 0;
      __syncthreads();
      row.template select<!WHOLE>(lo, hi, [&](int n) { return static_cast<int>(atomicAdd(&s.found32[1], static_cast<uint32_t>(n))); },
                 [&](int i, int at) {
                   if (at < kList) s.list[at] = i;
                 });
      __syncthreads();
      listed = s.found32[1];
      list_from = b0;
      if (listed > kList) return false;
      for (int at = tid; at < listed; at += kThreads) {
        const uint32_t i = s.list[at];
        s.list[at] = static_cast<uint64_t>(key_of(to_f32(row.x[i]))) << 32 | ~i;
      }
      __syncthreads();
      return true;
    };
    // The cut at the last of the list that is needed for counts or weights to reach the limit, from `above` on.  While
    // there are more than kRank, they are parted by how far they are from the largest, and the part with the cut is left: keys are
    // all but proportional to values where these differ by little, and equal ones are parted by their places.
    auto cut_list = [&](bool by_count, uint64_t above, uint64_t limit) __attribute__((always_inline)) {
      constexpr int N = kList / kThreads;
      uint64_t v[N], by[N];                           // of each: what it counts for
      int n = listed, mine = 0;                       // of the thread: those of the part
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int i = tid + e * kThreads;
        v[e] = i < n ? s.list[i] : 0;                // 0: none
        by[e] = by_count || !v[e] ? 1 : w(value_of(list_key(v[e])));
      }
      while (n > kRank) {
        constexpr uint64_t none = ~static_cast<uint64_t>(0);
        uint64_t hi = 0, lo = none;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          hi = larger(hi, v[e]);
          lo = smaller(lo, v[e] ? v[e] : none);
        }
#pragma unroll
        for (int off = 32; off; off >>= 1) {
          hi = larger(hi, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(hi), off, 64)));
          lo = smaller(lo, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(lo), off, 64)));
        }
        __syncthreads();
        if (lane == 0) s.ends[wave][0] = hi, s.ends[wave][1] = lo;
        for (int i = tid; i < kBins; i += kThreads) s.bin_weight[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
          hi = larger(hi, s.ends[i][0]);
          lo = smaller(lo, s.ends[i][1]);
        }
        const uint64_t span = hi - lo;
        const int shift = larger(0, 64 - __clzll(span | 1) - kBinBits);
        int part[N];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          part[e] = v[e] ? static_cast<int>((hi - v[e]) >> shift) : -1;
          if (v[e])
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.bin_weight[part[e]]),
                      static_cast<unsigned long long>(by[e]));
        }
        __syncthreads();
        uint64_t all;
        const uint64_t sum = tid < kBins ? s.bin_weight[tid] : 0;
        const uint64_t had = above + before64(sum, s, all);
        // the part that reaches the limit; where rounding leaves that behind all, the last that has any
        if (sum && had < limit && (had + sum >= limit || had + sum == above + all)) {
          s.found32[0] = tid;
          s.found64[0] = had;
        }
        mine = 0;
        __syncthreads();
        above = s.found64[0];
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (part[e] != static_cast<int>(s.found32[0])) v[e] = 0;
          mine += v[e] != 0;
        }
        n = static_cast<int>(sum64(mine, s));
      }
      // the left ones next to each other
      __syncthreads();
      if (tid == 0) s.found32[3] = 0, s.found64[1] = 0;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (v[e]) {
          const uint32_t at = atomicAdd(&s.found32[3], 1u);
          s.other[at] = v[e];
          s.rank_weight[at] = by[e];
        }
      __syncthreads();
      rank_all(s.other, n, s);
      if (tid < n) {
        const uint64_t had = above + s.rank_before[tid];
        if (had < limit && (had + s.rank_weight[tid] >= limit || s.rank[tid] + 1 == static_cast<uint32_t>(n))) s.found64[1] = s.other[tid];
      }
      __syncthreads();
      cut_key = list_key(s.found64[1]);
      cut_last = list_index(s.found64[1]);
    };
    // Where only the values are counted, a top_k that leaves all of them cuts at the last: they are few.
    const bool by_k = counts && (!weights || static_cast<uint64_t>(rules.top_k) < all);
    // Places are known to an eighth of a bin, and their edges exact, where they are not too far from zero; at temperatures over
    // 92 products of the smallest values round to 0, so that an edge there is far from its quotient.
    bool digits = !(fabsf(bins.base) < 0x1p20f && bins.scale >= 0.125f && bins.scale < INFINITY);
    // all up to the bin, where that fits a list, or the bin alone
    auto bring = [&](int b) __attribute__((always_inline)) { return gather(s.above_count[b] + s.bin_count[b] <= kList ? 0 : b, b); };
    uint64_t sum = total;
    int cut_bin = kBins;
    auto limit_of = [&](uint64_t sum) __attribute__((always_inline)) {
      return larger(static_cast<uint64_t>(ceil(static_cast<double>(rules.top_p) * static_cast<double>(sum))), static_cast<uint64_t>(1));
    };
    // All that may be kept, where it is few: one order gives every filter's cut, an order by place the token.
    auto draw_few = [&]() __attribute__((always_inline)) {
      const int n = listed;
      const uint64_t v = tid < n ? s.list[tid] : 0, wi = tid < n ? w(value_of(list_key(v))) : 0;
      if (tid < n) s.rank_weight[tid] = wi;
      rank_all(s.list, n, s);
      bool keep = tid < n;
      if (by_k) {
        keep &= tid < n && s.rank[tid] < static_cast<uint32_t>(rules.top_k);
        sum = sum64(keep ? wi : 0, s);
      }
      if (rules.top_p < 1.f) keep &= tid < n && s.rank_before[tid] < limit_of(sum);
      keep &= list_key(v) >= least;
      const uint64_t kept_sum = sum64(keep ? wi : 0, s);
      if (tid < n) {
        s.rank_weight[tid] = keep ? wi : 0;
        s.other[tid] = v << 32 | tid;                // by the index from the lowest up
      }
      __syncthreads();
      rank_all(s.other, n, s);
      const uint64_t target = pick(u, kept_sum);
      if (keep && s.rank_before[tid] <= target && s.rank_before[tid] + wi > target) *token = list_index(v);
    };
    const bool counted = counts && !weights;       // the chunks' weights are not known: the list has to hold all
    if (by_k && !digits) {
      const uint64_t k = smaller(static_cast<uint64_t>(rules.top_k), all);
      const int b = find_bin(s.above_count, k);
      digits = !bring(b) || (counted && list_from > 0);
      if (!digits) {
        if (list_from == 0 && listed <= kRank) return draw_few();
        cut_bin = b;
        cut_list(true, list_from ? s.above_count[list_from] : 0, k);
        if (rules.top_p < 1.f) {
          uint64_t mine = 0;
          for (int i = tid; i < listed; i += kThreads) {
            const uint32_t key = list_key(s.list[i]);
            if (key > cut_key || (key == cut_key && list_index(s.list[i]) <= cut_last)) mine += w(value_of(key));
          }
          sum = sum64(mine, s);
          if (list_from) sum += s.above_weight[list_from];
        }
      }
    }
    if (rules.top_p < 1.f && !digits) {
      const uint64_t limit = limit_of(sum);
      // at most the bin of top_k's cut, whose sum in the chunks' units may be a few less
      const int b = list_from == 0 ? 0 : smaller(find_bin(s.above_weight, limit), cut_bin);
      uint64_t above = 0;
      if (b < list_from) {
        // how many there are is known to a factor of 2^(11/8): a bin that cannot fit is not tried
        digits = (!WHOLE && s.bin_count[b] > kList * 2.6f) || !bring(b);
        if constexpr (!WHOLE) {
          if (digits) {
            float lo, hi;
            edges(b, b, lo, hi);
            listed = part_bin(row, w, s, key_of(lo), smaller(key_of(hi), top), least, s.above_weight[b], limit, a.by_chunk);
            list_from = b;
            above = s.found64[0];
            parted = true;
            digits = listed < 0;
          }
        }
      }
      if (!digits) {
        if (!by_k && !parted && list_from == 0 && listed <= kRank) return draw_few();
        if (list_from) cut_bin = b;
        if (!parted && list_from) above = s.above_weight[list_from];
        cut_list(false, above, limit);
      }
    }
    if (rules.min_p > 0.f && !digits) {
      // a weight of min_p is -8 log2(min_p) bins down, or next to that: all before the bin before it have more, all behind the
      // second after it less
      const int b = static_cast<int>(fminf(fmaxf(floorf(-8.f * static_cast<float>(power)) - 1.f, 0.f), kBins - 1));
      if (b < list_from) {
        const int end = smaller(smaller(b + 3, kBins - 1), cut_bin);
        const int begin = s.above_count[end] + s.bin_count[end] <= kList ? 0 : smaller(b, end);
        digits = !gather(begin, end);
        parted = false;
        if constexpr (!WHOLE) {
          if (digits) {                                // more than a list holds: what is kept of them goes to the chunks' sums at once
            float lo, hi;
            edges(begin, end, lo, hi);
            __syncthreads();
            if (tid < kChunks) s.chunk_sum[tid] = 0;
            __syncthreads();
            row.template select<false>(value_of(least), hi, [](int) { return 0; }, [&](int i, int) {
              const float x = to_f32(row.x[i]);
              if (kept(key_of(x), static_cast<uint32_t>(i)))
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.chunk_sum[fdiv(static_cast<uint32_t>(i), a.by_chunk)]),
                          static_cast<unsigned long long>(w(x)));
            });
            listed = 0;
            list_from = begin;
            parted = true;
            digits = false;
          }
        }
        if (!digits && !parted && begin == 0 && listed <= kRank && !by_k && !(rules.top_p < 1.f)) return draw_few();
      }
    }
    if (digits) {
      __syncthreads();
      return draw_by_digits(row, w, s, rules, top, least, u, token);
    }
  }

  // the chunk: what it has in bins that are kept, and of the list
  uint64_t chunk_sum = units(my_sum, my_shift);
  if (list_from < kBins) {
    __syncthreads();
    for (int i = tid; i < kChunks * 8; i += kThreads) s.other[i] = 0;      // chunks' sums, eight of each, so that atomics seldom meet
    __syncthreads();
    for (int i = tid; i < listed; i += kThreads) {
      const uint64_t v = s.list[i];
      if (!kept(list_key(v), list_index(v))) continue;
      atomicAdd(reinterpret_cast<unsigned long long*>(&s.other[fdiv(list_index(v), a.by_chunk) * 8 + (tid & 7)]),
                static_cast<unsigned long long>(w(value_of(list_key(v)))));
    }
    __syncthreads();
    if (tid < kChunks) {
      uint64_t sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += s.other[tid * 8 + i];
      s.chunk_sum[tid] = parted ? s.chunk_sum[tid] + sum : sum;
    }
    __syncthreads();
    if (list_from > 0)
      for (int c = wave; c < a.chunks; c += kWaves) {
        if (__shfl(my_top, c, 64) <= kNever) continue;
        const float off = __shfl(my_off, c, 64);
        const double shift = __shfl(my_shift, c, 64);
        uint64_t part = 0;
#pragma unroll
        for (int j = 0; j < kBins / 64; ++j) {
          const uint64_t v = chunks[c].weight[j * 64 + lane];
          if (static_cast<int>(fminf(j * 64 + lane + off, kBins - 1)) < list_from) part += units(v, shift);
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) part += __shfl_xor(static_cast<unsigned long long>(part), o, 64);
        if (lane == 0) s.chunk_sum[c] += part;
      }
    __syncthreads();
    chunk_sum = mine ? s.chunk_sum[lane] : 0;
  }
  uint64_t upto = chunk_sum;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t up = __shfl_up(static_cast<unsigned long long>(upto), off, 64);
    if (lane >= off) upto += up;
  }
  const uint64_t target = pick(u, __shfl(static_cast<unsigned long long>(upto), 63, 64));
  const uint64_t over = __ballot(upto > target);
  if (over == 0) {                                 // no sums at all
    if (tid == 0) *token = first;
    return;
  }
  const int c = smaller(__ffsll(static_cast<unsigned long long>(over)) - 1, a.chunks - 1);
  const uint64_t left = target - __shfl(static_cast<unsigned long long>(upto - chunk_sum), c, 64);
  // The token in the chunk: neighbouring values a thread, 8 of them (a longer chunk: 8 times a whole number) at a time.
  const int64_t lo = static_cast<int64_t>(c) * a.chunk, end = smaller(lo + a.chunk, static_cast<int64_t>(a.v));
  const int64_t run = (static_cast<int64_t>(a.chunk) + kThreads * 8 - 1) / (kThreads * 8) * 8, from = smaller(lo + tid * run, end), to = smaller(from + run, end);
  auto weights = [&](int64_t at, uint64_t(&v)[8]) __attribute__((always_inline)) {
    T x[8];
    if (at + 8 <= to) {
      __builtin_memcpy(x, row.x + at, sizeof x);       // at element alignment
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = at + e < to ? row.x[at + e] : from_f32<T>(-INFINITY);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = to_f32(x[e]);
      v[e] = kept(key_of(f), static_cast<uint32_t>(at + e)) ? w(f) : 0;
    }
  };
  uint64_t sum = 0, total, v[8];
  for (int64_t at = from; at < to; at += 8) {
    weights(at, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[e];
  }
  uint64_t start = before64(sum, s, total);
  // the chunk's own sum may differ in its last bits
  const uint64_t want = total ? smaller(left, total - 1) : 0;
  if (total == 0) {
    if (tid == 0) *token = first;
  } else if (start <= want && start + sum > want) {
    for (int64_t at = from; at < to && start <= want; at += 8) {
      if (run > 8) weights(at, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (start <= want && start + v[e] > want) *token = at + e;
        start += v[e];
      }
    }
  }
}

// Values of a chunk, and chunks of a row: 16 values a thread.  Smaller chunks add more bins up than they spread work (of 8192 and of 2048
// values: 128 rows of 100003 by top-p 62 and 89 us, 256 of 131072 unfiltered 48 and 137, one row of 131072 by top-p 38 and 46; only
// unfiltered it is 16 and 11).
int64_t chunk_of(const wc_sample_args& p) { return std::max<int64_t>(8192, cdiv(cdiv(p.v, kChunks), 16) * 16); }
int64_t chunks_of(const wc_sample_args& p) { return cdiv(p.v, chunk_of(p)); }

int32_t check(const wc_sample_args& p, const char* what) {
  WC_REQUIRE(dtype_size(p.dtype), WC_ERR_DTYPE, "%s: dtype %d", what, p.dtype);
  WC_REQUIRE(p.n >= 0 && p.m >= 0 && p.v >= 0, WC_ERR_SHAPE, "%s: negative size", what);
  WC_REQUIRE(p.v < (1ll << 30) && mul_sat({p.n, p.m}) < (1ll << 22) && mul_sat({p.n, p.m, std::max<int64_t>(chunks_of(p), 1)}) < (1ll << 23), WC_ERR_LIMIT,
             "%s: 2^30 logits of a row, 2^22 rows or 2^23 chunks of them, or more", what);
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
  if (check(*args, "wc_sample")) return -1;
  const int64_t chunks = chunks_of(*args);             // rows of one have their sums in LDS
  return chunks > 1 ? args->n * args->m * chunks * static_cast<int64_t>(sizeof(ChunkSums)) : 0;
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
  const int64_t need = wc_sample_workspace_bytes(args);
  WC_REQUIRE(need == 0 || (p.workspace && p.workspace_bytes >= need), WC_ERR_ARG, "%s: workspace of %lld bytes, %lld needed", what,
             (long long)p.workspace_bytes, (long long)need);
  WC_REQUIRE(aligned(p.workspace, 16), WC_ERR_ALIGN, "%s: workspace must be 16-byte aligned", what);
  a.sums = static_cast<ChunkSums*>(p.workspace);
  a.chunk = static_cast<int32_t>(chunk_of(p));
  a.chunks = static_cast<int32_t>(chunks_of(p));
  int bits = 0;
  while ((1ll << bits) < p.v) ++bits;
  a.fraction = std::min(48, 63 - bits);
  a.by_m = make_fastdiv(static_cast<uint32_t>(p.m));
  a.by_rows = make_fastdiv(static_cast<uint32_t>(p.x_rows_inner));
  a.by_chunks = make_fastdiv(static_cast<uint32_t>(a.chunks));
  a.by_chunk = make_fastdiv(static_cast<uint32_t>(a.chunk));
  const uint32_t rows = static_cast<uint32_t>(p.n * p.m);
  const hipStream_t s = as_stream(stream);
  auto go = [&](auto t) {
    typedef decltype(t) T;
    if (a.chunks == 1) {
      sample_rows_kernel<T, true><<<rows, kThreads, 0, s>>>(a);
    } else {
      sample_chunks_kernel<T><<<rows * static_cast<uint32_t>(a.chunks), kChunkThreads, 0, s>>>(a);
      sample_rows_kernel<T, false><<<rows, kThreads, 0, s>>>(a);
    }
  };
  if (p.dtype == WC_F32)
    go(float());
  else if (p.dtype == WC_BF16)
    go(bf16());
  else
    go(f16());
  return check_launch(what);
}
