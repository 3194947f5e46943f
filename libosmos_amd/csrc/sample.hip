// libosmos MI355X - osmos_sample (include/osmos_rows.h): one token for each row of logits.
//
// tokens are put into bins of their logits, 23 an octave of weight: y = logit x 23 log2(e) / T, bin rint(y), its weight
// 2^(y / 23). a bin's weights are summed as whole numbers of 2^-42 of its middle's weight, so that the sums do not depend on
// their order; a prefix of the tokens' order is whole bins and then some of one bin's tokens, which are found by their places: their
// logits' bits and indexes.
//
// a row is cut into slices: scan_kernel makes each slice's bins, plan_kernel adds a row's up and finds the bins that the limits and
// the token lie in, list_kernel lists these bins' tokens, draw_kernel chooses among them. bins are whole numbers of y, so that slices
// agree on them without knowing the row's maximum; a slice keeps the 1024 below its own. a short row is one kernel, its tokens in
// registers.
#include <type_traits>

#include "rowshost.h"
#include "common.h"
#include "lanes.h"

namespace osm {
namespace rows {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 1024;           // 44.5 octaves below the greatest weight: what is further down is in no bin
constexpr double kOctave = 23.0;
constexpr double kOne = 4398046511104.0;  // 2^42: 2^20 tokens of up to 2^(1 / 46) stay under 2^63
constexpr uint32_t kList = 2048;      // tokens that are looked at in LDS; more are looked for in the row each time
constexpr uint32_t kFew = 1024;       // a top_k up to this needs the weights of its own tokens alone: they are listed
constexpr uint32_t kCrowd = 64;       // tokens of a part that are compared with one another

// a logit as the order takes it: +infinity as the type's greatest value (a NaN stays one, and is greater than nothing)
template <uint32_t T> constexpr float kGreatest = T == OSMOS_F32 ? 3.40282346638528860e38f : T == OSMOS_F16 ? 65504.0f : 3.38953138925153547e38f;
template <uint32_t T>
__device__ inline float ordered(float x) {
  return x > kGreatest<T> ? kGreatest<T> : x;
}
template <uint32_t T>
__device__ inline float logit_at(const void* p, uint64_t i) {
  if constexpr (T == OSMOS_F32) return ordered<T>(gload<float>((const float*) p + i));
  else if constexpr (T == OSMOS_F16) return ordered<T>((float) gload<_Float16>((const _Float16*) p + i));
  else return ordered<T>((float) gload<__bf16>((const __bf16*) p + i));
}
// a token's place in the order (the greatest logit first, the lower index first among equals): the logit's bits, without those
// that are zero in all of type T's, above `bits` of its index
template <uint32_t T> constexpr int kDrop = T == OSMOS_F32 ? 0 : T == OSMOS_F16 ? 13 : 16;
template <uint32_t T>
struct Order {
  int bits;
  __device__ inline uint64_t place(float x, uint32_t i) const {
    const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
    return (uint64_t) ((b & 0x80000000u ? b : ~b & 0x7FFFFFFFu) >> kDrop<T>) << bits | i;
  }
  __device__ inline float logit(uint64_t place) const {
    const uint32_t k = (uint32_t) (place >> bits) << kDrop<T>;
    return __uint_as_float(k & 0x80000000u ? k : (~k & 0x7FFFFFFFu) >> kDrop<T> << kDrop<T>);
  }
  __device__ inline uint32_t index(uint64_t place) const { return (uint32_t) place & ((1u << bits) - 1); }
};

// 2^(f / 23) for -1/2 <= f <= 1/2, within 2^-45 (its series to the fifth power)
__device__ inline double part_weight(double f) {
  constexpr double c = 0.69314718055994530942 / kOctave;
  double k5 = c * c * c * c * c / 120, k4 = c * c * c * c / 24, k3 = c * c * c / 6, k2 = c * c / 2, k1 = c;
#if __HIP_DEVICE_COMPILE__
  asm("" : "+s"(k5), "+s"(k4), "+s"(k3), "+s"(k2), "+s"(k1));  // (in scalar registers: one instruction a step)
#endif
  double r = __builtin_fma(f, k5, k4);
  r = __builtin_fma(f, r, k3);
  r = __builtin_fma(f, r, k2);
  r = __builtin_fma(f, r, k1);
  return __builtin_fma(f, r, 1.0);
}
// the same as a whole number of 2^-42 (added to 2^52, whose last bit is 1)
__device__ inline uint64_t whole_weight(double f) {
  return (uint64_t) __double_as_longlong(__builtin_fma(part_weight(f), kOne, 4503599627370496.0)) - 0x4330000000000000ull;
}
__device__ inline uint64_t whole(double x) { return (uint64_t) __builtin_rint(x); }

struct SampleArgs {
  const void* logits;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  int32_t *token, *kept;
  float *prob, *probs;
  uint64_t stride;
  uint32_t n, vocab;
  uint32_t slices, slice;  // a row's, and a slice's tokens
  int bits;                // of a token's index
  uint8_t *parts, *plans, *cuts;  // the workspace: each slice's Part, each row's RowPlan and Drawn
};
// what a row asks for
struct Wish {
  float temperature, top_p, min_p, u;
  int32_t k;
  __device__ inline Wish(const SampleArgs& a, uint32_t t)
      : temperature(a.temperature ? a.temperature[t] : 1.0f), top_p(a.top_p ? a.top_p[t] : 1.0f), min_p(a.min_p ? a.min_p[t] : 0.0f), u(a.u[t]),
        k(a.top_k ? a.top_k[t] : 0) {}
};
// whether a row's bins need no weights: those of a few listed tokens do
__device__ inline bool few(int32_t k) { return k > 0 && (uint32_t) k <= kFew; }

// what is known of a slice
struct Part {
  uint64_t first;  // the place of its first token (its index in a greedy row alone); ~0: none
  double top;      // its first bin
  uint32_t valid;  // tokens that can be chosen; 0 for a greedy row too, and then no bins
  uint64_t mass[kBins];  // (unused for a few)
  uint32_t count[kBins];
};
// what a row was drawn from, for its probabilities
struct Drawn {
  uint64_t last;  // the last kept place; ~0: all
  double by, top, least_y, share;  // least_y: what a kept token's y is at least; share 0: the row's one token is `last`, or none
};

struct Sum {
  uint32_t n;  // tokens
  uint64_t m;  // their weights
};

// a row's limits and the bins that they and its token lie in
struct Plan {
  double by, top, part, draw, edge;  // Scale; top_p and u in their ranges; min_p as a y
  uint64_t all;             // the bins' weights
  uint32_t valid, listed;   // tokens that can be chosen, that are listed (more than kList: those past it are not)
  uint32_t k;               // top_k where it limits, or 0; k_bin kBins: among tokens of no weight
  int k_bin, m_bin;         // kBins: none
  int done, small, by_p;    // done: the row's token is given already; small: all bins up to to[0] are listed, whatever their weights
  int far;                  // min_p alone ends the kept tokens, and past the bins: those from there on are counted, into `past`
  uint32_t past;
  int split;                // a listed bin's parts, as a power of two
  int from[4], to[4], slot[4];  // the listed bins, apart from one another (kBins: none); how many are listed before a span's
  float low[4], high[4];    // these spans' logits, a little wide; low is finite: -infinity is no token, and stands past a row's end
};
// a row's bins' prefix sums: weights (of kOne the first bin's middle) and tokens
struct Prefix {
  uint64_t before[kBins + 1];
  uint32_t ahead[kBins + 1];
};
struct RowPlan {
  Plan plan;
  Prefix prefix;
  uint64_t list[kList];
};

struct ScanLds {
  uint64_t mass[kBins];
  uint32_t count[kBins];
  Sum wave[kSampleWaves];
  float greatest[kSampleWaves];
  uint32_t index;
};
constexpr int kValues = 8192;  // bf16: the values from 2^-24 to 2^8 of either sign
struct ValueLds : ScanLds {
  uint32_t value[kValues];
};
template <bool VALUES> using ScanOf = std::conditional_t<VALUES, ValueLds, ScanLds>;
struct PlanLds {
  Plan plan;
  Prefix prefix;
  Sum wave[kSampleWaves];
};
struct DrawLds {
  uint64_t part_m[kBins], part_lo[kBins], part_hi[kBins];  // sums of weights; least and greatest places
  uint32_t part_n[kBins], before_n[kBins], filled[kBins];
  uint64_t sorted[kList], weight[kList];  // a part's tokens together; then in order, and the weights up to each
  Sum wave[kSampleWaves];
  uint64_t word[kSampleWaves], found[4], sum;
  uint32_t at, crowded;
};
struct WholeLds : PlanLds {
  union {
    ScanLds scan;
    DrawLds draw;
  };
  uint64_t list[kList];
};

template <int STEP = 0>
__device__ inline Sum wave_sums(Sum x) {  // inclusive
  x.n += from_below<STEP>(x.n, 0u), x.m += from_below<STEP>(x.m, (uint64_t) 0);
  if constexpr (STEP < 5) return wave_sums<STEP + 1>(x);
  else return x;
}
template <int STEP = 0>
__device__ inline uint64_t wave_least(uint64_t x) {  // lane 63: of all
  const uint64_t y = from_below<STEP>(x, ~0ull);
  x = y < x ? y : x;
  if constexpr (STEP < 5) return wave_least<STEP + 1>(x);
  else return x;
}
template <int STEP = 0>
__device__ inline float wave_greatest(float x) {  // lane 63: of all
  x = fmaxf(x, __uint_as_float(from_below<STEP>(__float_as_uint(x), 0xFF800000u)));
  if constexpr (STEP < 5) return wave_greatest<STEP + 1>(x);
  else return x;
}
// inclusive sums over the workgroup's threads in their order
template <typename L>
__device__ inline Sum scan_sum(Sum x, L& l) {
  const int wave = threadIdx.x / 64;
  x = wave_sums(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) l.wave[wave] = x;
  __syncthreads();
  Sum w = {(threadIdx.x & 63) < kSampleWaves ? l.wave[threadIdx.x & 15].n : 0, (threadIdx.x & 63) < kSampleWaves ? l.wave[threadIdx.x & 15].m : 0};
  w = wave_sums(w);
  if (wave) {
    x.n += (uint32_t) __builtin_amdgcn_readlane((int) w.n, wave - 1);
    x.m += (uint64_t) (uint32_t) __builtin_amdgcn_readlane((int) (w.m >> 32), wave - 1) << 32 | (uint32_t) __builtin_amdgcn_readlane((int) w.m, wave - 1);
  }
  return x;
}
template <typename L>
__device__ inline Sum total(Sum x, L& l) {
  x = wave_sums(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) l.wave[threadIdx.x / 64] = x;
  __syncthreads();
  x = {0, 0};
#pragma unroll
  for (int w = 0; w < kSampleWaves; w++) x.n += l.wave[w].n, x.m += l.wave[w].m;
  return x;
}
template <typename L>
__device__ inline uint64_t least(uint64_t x, L& l) {
  x = wave_least(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) l.word[threadIdx.x / 64] = x;
  __syncthreads();
  x = l.word[0];
#pragma unroll
  for (int w = 1; w < kSampleWaves; w++) x = l.word[w] < x ? l.word[w] : x;
  return x;
}

// where a row's logits lie on the bins' scale
struct Scale {
  double by, top;  // bins a unit of logit; the first bin
  __device__ inline double y(float x) const { return (double) x * by; }
  __device__ inline int bin(double middle) const {  // kBins: none
    const double b = top - middle;
    return b < kBins ? (int) b : kBins;
  }
  __device__ inline int bin_of(float x) const { return bin(__builtin_rint(y(x))); }
};
__device__ inline double bins_a_unit(float temperature) { return kOctave * 1.4426950408889634074 / (double) temperature; }

// 16 bytes of logits at any address that their type allows, as they are (past the end: -infinity)
template <uint32_t T> constexpr uint32_t kPer = T == OSMOS_F32 ? 4 : 8;
typedef uint32_t u32x4_1 __attribute__((ext_vector_type(4), aligned(1)));
template <uint32_t T>
struct Piece {
  uint32_t w[4];
  __device__ inline void load(const void* p, uint32_t i, uint32_t end) {
    if (i + kPer<T> <= end) {
      const u32x4_1 v = gload<u32x4_1>((const uint8_t*) p + (uint64_t) i * kv::size_of(T));
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = v[j];
    } else if constexpr (T == OSMOS_F32) {
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) w[j] = i + j < end ? gload<uint32_t>((const uint32_t*) p + i + j) : 0xFF800000u;
    } else {
      constexpr uint32_t none = T == OSMOS_F16 ? 0xFC00u : 0xFF80u;
#pragma unroll
      for (uint32_t j = 0; j < 4; j++)
        w[j] = (i + 2 * j < end ? (uint32_t) gload<uint16_t>((const uint16_t*) p + i + 2 * j) : none) |
               (i + 2 * j + 1 < end ? (uint32_t) gload<uint16_t>((const uint16_t*) p + i + 2 * j + 1) : none) << 16;
    }
  }
  __device__ inline float at(uint32_t j) const {
    if constexpr (T == OSMOS_F32) return __uint_as_float(w[j]);
    else if constexpr (T == OSMOS_BF16) return __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
    else return __half2float(__ushort_as_half((unsigned short) (w[j / 2] >> 16 * (j & 1))));
  }
};

// tokens begin .. end - 1 of a row, P pieces a thread and round (the rounds' loads in flight together)
template <uint32_t T, int P, uint32_t N = kSampleThreads>
struct Tokens {
  const void* p;
  uint32_t begin, end;
  static constexpr uint32_t kRound = N * kPer<T> * P;
  Piece<T> x[P];
  __device__ inline void load(uint32_t at) {
#pragma unroll
    for (int k = 0; k < P; k++) x[k].load(p, at + (k * N + threadIdx.x) * kPer<T>, end);
  }
  template <typename F>
  __device__ inline void loaded(uint32_t at, F f) const {
#pragma unroll
    for (int k = 0; k < P; k++)
#pragma unroll
      for (uint32_t j = 0; j < kPer<T>; j++) f(x[k].at(j), at + (k * N + threadIdx.x) * kPer<T> + j);
  }
  // those of a plan's spans' logits: most threads have none, so they are read again (what a piece has past the end is -infinity, less
  // than any low)
  template <typename F>
  __device__ inline void loaded_between(uint32_t at, const Plan& p, F f) const {
    const float l0 = p.low[0], h0 = p.high[0], l1 = p.low[1], h1 = p.high[1], l2 = p.low[2], h2 = p.high[2], l3 = p.low[3], h3 = p.high[3];
    const int spans = l3 <= h3 ? 4 : l2 <= h2 ? 3 : l1 <= h1 ? 2 : 1;
    uint32_t hits = 0;
    auto test = [&](auto in) __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < P; k++)
#pragma unroll
        for (uint32_t j = 0; j < kPer<T>; j++) hits = hits + hits + in(x[k].at(j));  // (the first one's bit the highest)
    };
    static_assert(P * kPer<T> <= 32);
    // (& and |: as && and || each comparison is a branch, 13 instructions a bf16 token in all instead of 11)
    if (spans == 1) test([&](float v) { return (v >= l0) & (v <= h0); });
    else if (spans == 2) test([&](float v) { return ((v >= l0) & (v <= h0)) | ((v >= l1) & (v <= h1)); });
    else test([&](float v) { return ((v >= l0) & (v <= h0)) | ((v >= l1) & (v <= h1)) | ((v >= l2) & (v <= h2)) | ((v >= l3) & (v <= h3)); });
    while (hits) {
      const uint32_t h = P * kPer<T> - 1 - __builtin_ctz(hits);
      hits &= hits - 1;
      const uint32_t i = at + (h / kPer<T> * N + threadIdx.x) * kPer<T> + h % kPer<T>;
      f(logit_at<T>(this->p, i), i);
    }
  }
  // all, where the first round is loaded: a second one is read again
  template <typename F>
  __device__ inline void again(F f) {
    if (end - begin <= kRound) loaded(begin, f);
    else each(f);
  }
  // in ascending order of a thread's own tokens
  template <typename F>
  __device__ inline void each(F f) {
    for (uint32_t at = begin; at < end; at += kRound) {
      load(at);
      loaded(at, f);
    }
  }
};

// the tokens that a row's choice can hang on: the listed ones where the list holds them, or all
template <uint32_t T>
struct Near {
  Tokens<T, 2> row;
  const Order<T>& order;
  const uint64_t* list;
  uint32_t n;
  template <typename F>
  __device__ inline void each(F f) {
    if (n <= kList)
      for (uint32_t i = threadIdx.x; i < n; i += kSampleThreads) f(order.logit(list[i]), order.index(list[i]));
    else
      row.each([&](float x, uint32_t i) {
        x = ordered<T>(x);
        if (x > -__builtin_inff()) f(x, i);
      });
  }
};

// a slice's first place and, but for a greedy row, its bins (into l.count and, unless k is small, l.mass): its tokens are one round, but
// by VALUES. bf16's tokens are few values, often: by VALUES they are counted by value, two a word, and each value is put into its bin
// once
template <uint32_t T, bool VALUES, typename R, typename L>
__device__ inline void scan_slice(R& row, const Order<T>& order, float temperature, int32_t k, L& l, uint64_t& first, double& top, uint32_t& valid) {
  constexpr uint32_t kLeastBits = 0x3380, kSpan = kValues / 2;  // (2^-24; the first and the last of the span stand for what is outside)
  const uint32_t tid = threadIdx.x;
  const float none = -__builtin_inff();
  const bool warm = temperature > 0.0f, mass = !few(k);
  row.load(row.begin);
  l.mass[tid] = 0, l.count[tid] = 0;
  if (tid == 0) l.index = ~0u;
  float best = none;
  uint32_t outside = 0;  // whether some of bf16's are not among its values
  if constexpr (VALUES) {
#pragma unroll
    for (int i = 0; i < kValues; i += kSampleThreads) l.value[i + tid] = 0;
    __syncthreads();
    for (uint32_t round = row.begin;;) {
#pragma unroll
      for (uint32_t k = 0; k < sizeof(row.x) / sizeof(row.x[0]); k++) {
        if (round + (k * kSampleThreads + tid) * kPer<T> >= row.end) break;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
          const uint32_t w = row.x[k].w[i], size = w & 0x7FFF7FFFu;
          u16x2 v = __builtin_bit_cast(u16x2, size);
          v = __builtin_elementwise_min(__builtin_elementwise_max(v, u16x2{kLeastBits, kLeastBits}), u16x2{kLeastBits + kSpan - 1, kLeastBits + kSpan - 1}) -
              u16x2{kLeastBits, kLeastBits};
          const uint32_t at = __builtin_bit_cast(uint32_t, v) << 2 | (w >> 1 & 0x40004000u);  // (4096 values of 4 bytes a sign)
          atomicAdd((uint32_t*) ((uint8_t*) l.value + (at & 0xFFFF)), 1u);
          atomicAdd((uint32_t*) ((uint8_t*) l.value + (at >> 16)), 1u);
        }
      }
      if ((round += row.kRound) >= row.end) break;
      row.load(round);
    }
    __syncthreads();
    // (what a last, partial piece has past the end is in the last)
    outside = l.value[0] | l.value[kSpan - 1] | l.value[kSpan] | (l.value[kValues - 1] - (row.begin - row.end) % kPer<T>);
    if (outside) {
      row.again([&](float x, uint32_t) { best = fmaxf(best, x); });
    } else {
#pragma unroll
      for (int j = 0; j < kValues / kSampleThreads; j++) {
        const uint32_t i = tid + j * kSampleThreads;
        if (l.value[i]) best = fmaxf(best, __uint_as_float((i % kSpan + kLeastBits) << 16 | i / kSpan << 31));
      }
    }
  } else {
    row.loaded(row.begin, [&](float x, uint32_t) { best = fmaxf(best, x); });
  }
  float most = wave_greatest(best);
  if ((tid & 63) == 63) l.greatest[tid / 64] = most;
  __syncthreads();
  most = l.greatest[0];
#pragma unroll
  for (int w = 1; w < kSampleWaves; w++) most = fmaxf(most, l.greatest[w]);
  most = ordered<T>(most);
  first = ~0ull, top = 0.0, valid = 0;
  if (!(most > none)) return;
  if (!warm) {  // (the lowest index among equals; elsewhere its logit is all that is asked for)
    uint32_t at = ~0u;
    row.again([&](float x, uint32_t i) { at = ordered<T>(x) == most && i < at ? i : at; });
    if (at != ~0u) atomicMin(&l.index, at);
    __syncthreads();
    first = order.place(most, l.index);
    return;
  }
  first = order.place(most, 0);
  Scale sc = {bins_a_unit(temperature), 0.0};
  sc.top = top = __builtin_rint(sc.y(most));
  auto add = [&](float x, uint32_t n, bool mass) __attribute__((always_inline)) {
    x = ordered<T>(x);
    const double y = sc.y(x), middle = __builtin_rint(y), b = sc.top - middle;
    if (b < kBins) {
      const int i = (int) b;
      atomicAdd(&l.count[i], n);
      if (mass) atomicAdd((unsigned long long*) &l.mass[i], (unsigned long long) (n * whole_weight(y - middle)));
    } else {
      valid += x > none ? n : 0;
    }
  };
  if constexpr (VALUES) {
    if (outside)
      row.again([&](float x, uint32_t) {
        const uint32_t v = (__float_as_uint(x) >> 16 & 0x7FFF) - kLeastBits;
        if ((int) v < 1 || v >= kSpan - 1) add(x, 1, mass);
      });
#pragma unroll
    for (int j = 0; j < kValues / kSampleThreads; j++) {
      const uint32_t i = tid + j * kSampleThreads, n = l.value[i];
      if (n && i % kSpan && i % kSpan != kSpan - 1) add(__uint_as_float((i % kSpan + kLeastBits) << 16 | i / kSpan << 31), n, mass);
    }
  } else {
    if (mass) row.loaded(row.begin, [&](float x, uint32_t) { add(x, 1, true); });
    else row.loaded(row.begin, [&](float x, uint32_t) { add(x, 1, false); });
  }
  __syncthreads();
  valid = total(Sum{valid + l.count[tid], 0}, l).n;
}

// 16 bytes of a slice a thread and round, and of a row that is one slice
template <uint32_t T, bool VALUES> constexpr int kPieces = VALUES ? 4 : 16 / kPer<T>;
template <uint32_t T> constexpr int kRowPieces = 32 / kPer<T>;
// bound by its vector and LDS instructions: in all 33 and 3 a token, of which two are atomics (48 rows of 151001 floats 14.5 us); by value
// 12 and 1.8 (256 rows of 129024 bf16 25.3 us; token by token the call takes 16 us more)
template <uint32_t T, bool VALUES>
__global__ __launch_bounds__(kSampleThreads, 8) void scan_kernel(SampleArgs a) {
  __shared__ ScanOf<VALUES> l;
  const uint32_t t = blockIdx.x / a.slices, s = blockIdx.x - t * a.slices, begin = s * a.slice, tid = threadIdx.x;
  const uint32_t end = begin + a.slice < a.vocab ? begin + a.slice : a.vocab;
  Tokens<T, kPieces<T, VALUES>> row = {(const uint8_t*) a.logits + t * a.stride * kv::size_of(T), begin, end};
  Part* part = (Part*) a.parts + blockIdx.x;
  const Order<T> order = {a.bits};
  const int32_t k = a.top_k ? a.top_k[t] : 0;
  uint64_t first;
  double top;
  uint32_t valid;
  scan_slice<T, VALUES>(row, order, a.temperature ? a.temperature[t] : 1.0f, k, l, first, top, valid);
  if (valid) {
    part->count[tid] = l.count[tid];
    if (!few(k)) part->mass[tid] = l.mass[tid];
  }
  if (tid == 0) part->first = first, part->top = top, part->valid = valid;
}

// 2^(-i / 23), and a bin's weight by the first's
__constant__ double kRoots[23] = {1.0, 0.9703127527497981, 0.9415068381488909, 0.913556091857009, 0.886435126281122, 0.8601193075159503, 0.834584732969052, 0.809808209650156, 0.7857672331050286, 0.7624399669747326, 0.739805223161718, 0.7178424425847253, 0.6965316765050238, 0.6758535684070215, 0.655789336416791, 0.63632075624254, 0.6174301446215323, 0.599100343258425, 0.5813147032404313, 0.5640570699151549, 0.5473117682173594, 0.5310635884313455, 0.5152977723760047};
__device__ inline double bin_scale(int b) {
  const int o = b / 23;
  return ldexp(kRoots[b - 23 * o], -o);
}
// the weight that the first `part` of m's reach, and the one that the sum of the token drawn by `u` reaches
__device__ inline uint64_t p_goal(double part, uint64_t m) {
  const double g = __builtin_ceil((double) m * part);
  return g > 1.0 ? (uint64_t) g < m ? (uint64_t) g : m : 1;
}
__device__ inline uint64_t u_goal(double u, uint64_t m) {
  const uint64_t g = (uint64_t) __builtin_floor((double) m * u) + 1;
  return g < m ? g : m;
}

// a row's plan from its bins (thread i bin i's sums), by one wave after the sums: the others would only repeat it (6.6 us a row, so 2.5).
// what is written is there for all threads when it returns
template <uint32_t T>
__device__ inline void make_plan(const SampleArgs& a, uint32_t t, const Wish& wish, const Order<T>& order, PlanLds& l, uint64_t first, double top,
                                 uint32_t valid, Sum bin) {
  const uint32_t tid = threadIdx.x;
  const float temperature = wish.temperature, top_p = wish.top_p, min_p = wish.min_p, u = wish.u;
  const int32_t k = wish.k;
  const Scale sc = {bins_a_unit(temperature), top};
  Plan& p = l.plan;
  if (first == ~0ull || !(temperature > 0.0f)) {
    const bool none = first == ~0ull;
    if (tid == 0) {
      a.token[t] = none ? -1 : (int32_t) order.index(first);
      if (a.prob) a.prob[t] = none ? 0.0f : 1.0f;
      if (a.kept) a.kept[t] = none ? 0 : 1;
      if (a.probs) ((Drawn*) a.cuts)[t] = Drawn{first, 0.0, 0.0, 0.0, 0.0};
      p.done = 1;
    }
    __syncthreads();
    return;
  }
  const bool small = few(k);
  const Sum sum = scan_sum(Sum{bin.n, small ? 0 : whole((double) bin.m * bin_scale(tid))}, l);
  l.prefix.ahead[tid + 1] = sum.n, l.prefix.before[tid + 1] = sum.m;
  if (tid == 0) l.prefix.ahead[0] = 0, l.prefix.before[0] = 0;
  __syncthreads();
  if (tid < 64) {  // (one wave: the others would only repeat it)
    const uint32_t* ahead = l.prefix.ahead;
    const uint64_t *before = l.prefix.before, all = before[kBins];
    // the bin whose sum reaches `goal`, the ones before it not
    auto reaches = [&](const auto* sums, auto goal) {
      const uint64_t a = __ballot(sums[(tid + 1) * 16] >= goal);
      const int s = a ? __builtin_ctzll(a) : 63;
      const uint64_t b = __ballot(sums[s * 16 + (tid & 15) + 1] >= goal);
      return s * 16 + (b ? __builtin_ctzll(b) : 15);
    };
    const uint32_t limit = k > 0 && (uint32_t) k < valid ? k : 0;
    const bool by_k = limit && limit <= ahead[kBins], by_p = top_p < 1.0f;
    const double edge = sc.y(order.logit(first)) + (min_p > 0.0f ? kOctave * log2((double) (min_p < 1.0f ? min_p : 1.0f)) : 0.0);
    const int m_bin = min_p > 0.0f ? sc.bin(__builtin_rint(edge)) : kBins;
    const double part = top_p > 0.0f ? top_p : 0.0f, drawn = u > 0.0f ? u < 1.0f ? u : 0.99999994f : 0.0f;
    const int k_bin = by_k ? reaches(ahead, limit) : kBins;
    // the spans of bins that the token, top_p, top_k and min_p lie in
    int f[4] = {0, kBins, kBins, kBins}, g[4] = {by_k ? k_bin : kBins - 1, -1, -1, -1};
    if (!small) {
      uint64_t least_m = all, most_m = all;
      // (tokens of less than 2^-43 of the greatest's weight add nothing to a sum: a bin's tokens may end where they begin)
      if (by_k) f[2] = g[2] = k_bin, least_m = before[k_bin] > 1 ? before[k_bin] : 1, most_m = before[k_bin + 1];
      if (by_p) {
        f[1] = reaches(before, p_goal(part, least_m));
        g[1] = least_m == most_m ? f[1] : reaches(before, p_goal(part, most_m));
        least_m = before[f[1]] + 1, most_m = before[g[1] + 1];
      }
      if (m_bin < kBins) {
        f[3] = g[3] = m_bin;
        const uint64_t lo = before[m_bin] > 1 ? before[m_bin] : 1, hi = before[m_bin + 1];
        least_m = lo < least_m ? lo : least_m, most_m = hi < most_m ? hi : most_m;
      }
      f[0] = reaches(before, u_goal(drawn, least_m));
      g[0] = least_m == most_m ? f[0] : reaches(before, u_goal(drawn, most_m));
    }
    // in ascending order, spans that touch as one
    auto sort = [&](int i, int j) {
      const bool swap = f[j] < f[i];
      const int a0 = swap ? f[j] : f[i], a1 = swap ? g[j] : g[i], b0 = swap ? f[i] : f[j], b1 = swap ? g[i] : g[j];
      f[i] = a0, g[i] = a1, f[j] = b0, g[j] = b1;
    };
    if (!small) sort(0, 1), sort(2, 3), sort(0, 2), sort(1, 3), sort(1, 2);
    int from[4] = {f[0], kBins, kBins, kBins}, to[4] = {g[0], kBins, kBins, kBins}, last = 0;
#pragma unroll
    for (int i = 1; i < 4; i++) {
      if (f[i] >= kBins) continue;
#pragma unroll
      for (int n = 3; n >= 0; n--) {
        if (n != last) continue;
        if (f[i] <= to[n] + 1) to[n] = g[i] > to[n] ? g[i] : to[n];
        else if (n < 3) from[n + 1 < 4 ? n + 1 : 3] = f[i], to[n + 1 < 4 ? n + 1 : 3] = g[i], last = n + 1;
      }
    }
    int slots = 0, slot[4];
#pragma unroll
    for (int n = 0; n < 4; n++) slot[n] = slots, slots += from[n] < kBins ? to[n] - from[n] + 1 : 0;
    // (tokens past the bins add nothing to a sum: a min_p there says only how many of them are kept, which top_p or a top_k in the bins
    // settles by itself. such a plan's one span is the token's, and the fourth has the logits between the bins and the edge)
    const bool far = a.kept && min_p > 0.0f && m_bin == kBins && !by_p && k_bin == kBins;
    if (tid < 4) {
      const int a0 = tid == 0 ? from[0] : tid == 1 ? from[1] : tid == 2 ? from[2] : from[3], a1 = tid == 0 ? to[0] : tid == 1 ? to[1] : tid == 2 ? to[2] : to[3];
      const bool beyond = far && tid == 3, none = a0 >= kBins && !beyond;
      const double unit = 1.0 / sc.by, lo = (beyond ? edge : top - a1 - 0.5) * unit, hi = (top - a0 + 0.5) * unit;
      const float fl = (float) (lo - 1e-6 * fabs(lo) - 3e-45), fh = (float) (hi + 1e-6 * fabs(hi) + 3e-45);  // (two of float's least steps)
      p.from[tid] = a0, p.to[tid] = a1, p.slot[tid] = tid == 0 ? slot[0] : tid == 1 ? slot[1] : tid == 2 ? slot[2] : slot[3];
      p.low[tid] = none ? __builtin_inff() : fl > -kGreatest<T> ? fl : -kGreatest<T>;
      p.high[tid] = none ? -__builtin_inff() : fh < kGreatest<T> ? fh : __builtin_inff();
    }
    if (tid == 0) {
      p.by = sc.by, p.top = top, p.part = part, p.draw = drawn, p.edge = edge;
      p.all = all, p.valid = valid, p.listed = 0, p.k = limit, p.k_bin = k_bin, p.m_bin = m_bin;
      p.done = 0, p.small = small, p.by_p = by_p, p.far = far, p.past = 0;
      p.split = small ? 0 : 10 - (slots > 1 ? 32 - __builtin_clz(slots - 1) : 0);
    }
  }
  __syncthreads();
}

constexpr uint32_t kSlice = 16384, kValueSlice = 32768, kMostSlices = OSMOS_SAMPLE_MAX_VOCAB / kSlice;
constexpr int kAtOnce = 8;  // slices whose bins are loaded together
template <uint32_t T>
__global__ __launch_bounds__(kSampleThreads) void plan_kernel(SampleArgs a) {
  __shared__ PlanLds l;
  __shared__ double tops[kMostSlices];  // (every wave writes the same)
  const uint32_t t = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const Part* parts = (const Part*) a.parts + (uint64_t) t * a.slices;
  const Wish wish(a, t);
  const bool small = few(wish.k);
  // the slices' bins as they lie, while their tops are on the way (what a slice of no bins holds is left out): then each to its place
  uint32_t n[kAtOnce];
  uint64_t m[kAtOnce];
  auto load = [&](uint32_t s0) {
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const Part* from = parts + (s0 + i < a.slices ? s0 + i : s0);
      n[i] = from->count[tid], m[i] = small ? 0 : from->mass[tid];
    }
  };
  load(0);
  l.prefix.before[tid] = 0, l.prefix.ahead[tid] = 0;
  uint64_t first = ~0ull;
  double top = -__builtin_inf();
  uint32_t valid = 0;
  for (uint32_t s = lane; s < a.slices; s += 64) {  // (a lane a slice)
    const uint64_t f = parts[s].first;
    const uint32_t v = parts[s].valid;
    const double own = v ? parts[s].top : -__builtin_inf();
    tops[s] = own;
    top = fmax(top, own), valid += v;
    first = f < first ? f : first;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const uint64_t f = (uint64_t) (uint32_t) __shfl_xor((int) (first >> 32), o) << 32 | (uint32_t) __shfl_xor((int) first, o);
    first = f < first ? f : first;
    top = fmax(top, __shfl_xor(top, o));
    valid += (uint32_t) __shfl_xor((int) valid, o);
  }
  __syncthreads();
  for (uint32_t s0 = 0;;) {
#pragma unroll
    for (int i = 0; i < kAtOnce; i++) {
      const double b = s0 + i < a.slices ? top - tops[s0 + i] + (int) tid : kBins;  // (a slice of no bins: infinite)
      if (b < kBins) {
        atomicAdd(&l.prefix.ahead[(int) b], n[i]);
        atomicAdd((unsigned long long*) &l.prefix.before[(int) b], (unsigned long long) m[i]);
      }
    }
    if ((s0 += kAtOnce) >= a.slices) break;
    load(s0);
  }
  __syncthreads();
  const Sum bin = {l.prefix.ahead[tid], l.prefix.before[tid]};
  const Order<T> order = {a.bits};
  make_plan<T>(a, t, wish, order, l, first, top, valid, bin);
  RowPlan* to = (RowPlan*) a.plans + t;
  if (tid < sizeof(Plan) / 4) ((uint32_t*) &to->plan)[tid] = ((const uint32_t*) &l.plan)[tid];
  if (l.plan.done) return;
  to->prefix.before[tid + 1] = l.prefix.before[tid + 1], to->prefix.ahead[tid + 1] = l.prefix.ahead[tid + 1];
  if (tid == 0) to->prefix.before[0] = 0, to->prefix.ahead[0] = 0;
}

// a listed bin's number among them; -1: not listed
__device__ inline int slot_of(const Plan& p, int b) {
  int slot = -1;
#pragma unroll
  for (int i = 0; i < 4; i++) slot = b >= p.from[i] && b <= p.to[i] ? p.slot[i] + b - p.from[i] : slot;
  return b < kBins ? slot : -1;
}
// whether a token is of the plan's bins; one past all bins that min_p keeps is counted
__device__ inline bool planned(const Plan& p, float x, uint32_t& past) {
  const Scale sc = {p.by, p.top};
  const int b = sc.bin_of(x);
  if (p.far && b == kBins && sc.y(x) >= p.edge) past++;
  return slot_of(p, b) >= 0;
}

// the planned bins' tokens of a row, in any order: 48 rows of 151001 floats 8.4 us, 256 of 129024 bf16 16.2 (4.1 TB/s)
constexpr int kListThreads = 256, kListPieces = 4;
template <uint32_t T>
__global__ __launch_bounds__(kListThreads) void list_kernel(SampleArgs a, uint32_t blocks) {
  __shared__ uint64_t list[kList];
  __shared__ uint32_t listed, start, past;
  constexpr uint32_t each = kListThreads * kPer<T> * kListPieces;
  const uint32_t t = blockIdx.x / blocks, begin = (blockIdx.x - t * blocks) * each;
  RowPlan* row_plan = (RowPlan*) a.plans + t;
  Tokens<T, kListPieces, kListThreads> row = {(const uint8_t*) a.logits + t * a.stride * kv::size_of(T), begin,
                                          begin + each < a.vocab ? begin + each : a.vocab};
  row.load(begin);
  const Plan p = row_plan->plan;
  if (p.done) return;
  const Order<T> order = {a.bits};
  if (threadIdx.x == 0) listed = 0, past = 0;
  __syncthreads();
  uint32_t own_past = 0;
  row.loaded_between(begin, p, [&](float x, uint32_t i) {
    if (!planned(p, x, own_past)) return;
    const uint32_t at = atomicAdd(&listed, 1u);
    if (at < kList) list[at] = order.place(x, i);
  });
  if (own_past) atomicAdd(&past, own_past);
  __syncthreads();
  if (threadIdx.x == 0 && past) atomicAdd(&row_plan->plan.past, past);
  if (!listed) return;
  if (threadIdx.x == 0) start = atomicAdd(&row_plan->plan.listed, listed);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < listed && i < kList; i += kListThreads)
    if (start + i < kList) row_plan->list[start + i] = list[i];
}

struct Cut {
  uint64_t place;  // the last token
  uint32_t n;      // how many tokens up to it
  uint64_t m;      // their weights
};

// the first token of bin b with at least `rank` tokens of the bin up to it (MASS: with at least `goal` of weight up to it): a
// thousandth of what is left each time
template <uint32_t T, bool MASS>
__device__ Cut find(Near<T>& row, const Scale& sc, const Prefix& prefix, DrawLds& l, int b, uint32_t rank, uint64_t goal) {
  const double scale = bin_scale(b);
  const uint64_t before = prefix.before[b];
  const uint32_t tid = threadIdx.x;
  uint64_t lo = ~0ull, hi = ~0ull;  // (hi: the greatest place, inverted)
  row.each([&](float x, uint32_t i) {
    if (sc.bin_of(x) != b) return;
    const uint64_t at = row.order.place(x, i);
    lo = at < lo ? at : lo, hi = ~at < hi ? ~at : hi;
  });
  lo = least(lo, l), hi = ~least(hi, l);
  Sum base = {0, 0};
  for (int level = 0; level < 6; level++) {  // (a place has 52 bits)
    const int bits = hi > lo ? 64 - __builtin_clzll(hi - lo) : 0, shift = bits > 10 ? bits - 10 : 0;
    __syncthreads();
    l.part_n[tid] = 0, l.part_m[tid] = 0, l.part_lo[tid] = ~0ull, l.part_hi[tid] = 0;
    __syncthreads();
    row.each([&](float x, uint32_t i) {
      const double y = sc.y(x), middle = __builtin_rint(y);
      if (sc.bin(middle) != b) return;
      const uint64_t at = row.order.place(x, i);
      if (at < lo || at > hi) return;
      const uint32_t j = (uint32_t) ((at - lo) >> shift);
      atomicAdd(&l.part_n[j], 1u);
      atomicAdd((unsigned long long*) &l.part_m[j], (unsigned long long) whole_weight(y - middle));
      atomicMin((unsigned long long*) &l.part_lo[j], (unsigned long long) at);
      atomicMax((unsigned long long*) &l.part_hi[j], (unsigned long long) at);
    });
    __syncthreads();
    const Sum own = {l.part_n[tid], l.part_m[tid]};
    Sum sum = scan_sum(own, l);
    sum.n += base.n, sum.m += base.m;
    const Sum past = {sum.n - own.n, sum.m - own.m};
    const bool here = MASS ? before + whole((double) sum.m * scale) >= goal && before + whole((double) past.m * scale) < goal
                           : sum.n >= rank && past.n < rank;
    if (here) {
      const bool one = own.n == 1;
      l.found[0] = l.part_lo[tid], l.found[1] = one ? l.part_lo[tid] : l.part_hi[tid];
      l.found[2] = one ? sum.n : past.n, l.found[3] = one ? sum.m : past.m;
    }
    __syncthreads();
    lo = l.found[0], hi = l.found[1];
    base.n = (uint32_t) l.found[2], base.m = l.found[3];
    if (lo >= hi) break;
  }
  return Cut{lo, prefix.ahead[b] + base.n, before + whole((double) base.m * scale)};
}

// bins of more tokens than the list or a part holds, or limits that leave a bound over many bins: one by one, each bin looked
// through as often as it takes, by one workgroup a row: 64 rows of 128256 floats (normal, deviation 1.5), top_p 0.9, are 44 us at a
// temperature of 0.7 and 201 at 1.5, where the limits' bins hold some 2500 tokens; of 262144 (2.5), top_p 0.95, 55 and 363
template <uint32_t T>
__device__ __attribute__((noinline)) void draw_slowly(const void* logits, uint32_t vocab, const Order<T>& order, const Plan& p, Prefix& prefix,
                                                      const uint64_t* list, DrawLds& l, Cut& cut, Cut& d, double& least_y) {
  const uint32_t tid = threadIdx.x;
  const Scale sc = {p.by, p.top};
  Near<T> near = {{logits, 0, vocab}, order, list, p.listed};
  uint64_t all = p.all;
  if (p.small) {  // (the bins' weights are not known yet)
    l.part_m[tid] = 0;
    __syncthreads();
    near.each([&](float x, uint32_t) {
      const double y = sc.y(x), middle = __builtin_rint(y);
      const int b = sc.bin(middle);
      if (b < kBins && b <= p.to[0]) atomicAdd((unsigned long long*) &l.part_m[b], (unsigned long long) whole_weight(y - middle));
    });
    __syncthreads();
    const Sum sum = scan_sum(Sum{0, whole((double) l.part_m[tid] * bin_scale(tid))}, l);
    prefix.before[tid + 1] = sum.m;
    __syncthreads();
    all = prefix.before[kBins];
  }
  auto by_mass = [&](uint64_t goal) {
    if (prefix.before[tid + 1] >= goal && prefix.before[tid] < goal) l.at = tid;
    __syncthreads();
    const int b = (int) l.at;
    const Cut c = find<T, true>(near, sc, prefix, l, b, 0, goal);
    __syncthreads();
    return c;
  };
  cut = Cut{~0ull, p.k ? p.k : p.valid, all};
  if (p.k_bin < kBins) {
    cut = find<T, false>(near, sc, prefix, l, p.k_bin, p.k - prefix.ahead[p.k_bin], 0);
    __syncthreads();
  }
  if (p.by_p) cut = by_mass(p_goal(p.part, cut.m));
  if (p.m_bin < kBins) {
    Sum in = {0, 0};
    near.each([&](float x, uint32_t) {
      const double y = sc.y(x), middle = __builtin_rint(y);
      if (y >= p.edge && sc.bin(middle) == p.m_bin) in.n++, in.m += whole_weight(y - middle);
    });
    in = total(in, l);
    in = {prefix.ahead[p.m_bin] + in.n, prefix.before[p.m_bin] + whole((double) in.m * bin_scale(p.m_bin))};
    if (in.n < cut.n) cut.n = in.n, cut.m = in.m, least_y = p.edge;
  }
  d = by_mass(u_goal(p.draw, cut.m));
}

// the choice among the listed tokens: each one's count and weight up to it. a token's bin is cut into 2^split parts of places, each
// part has its tokens together, and each token is compared with the others of its part. at: the list's tokens tid and tid + 1024
template <uint32_t T>
__device__ inline void draw(const SampleArgs& a, uint32_t t, const Order<T>& order, const Plan& p, Prefix& prefix, const uint64_t* list,
                            uint64_t (&at)[2], DrawLds& l) {
  const uint32_t tid = threadIdx.x, n = p.listed;
  const void* logits = (const uint8_t*) a.logits + t * a.stride * kv::size_of(T);
  const Scale sc = {p.by, p.top};
  const bool small = p.small;
  if (tid < 4) l.found[tid] = 0;
  if (tid == 0) l.crowded = n > kList, l.at = 0;
  l.part_n[tid] = 0, l.part_m[tid] = 0, l.filled[tid] = 0, l.part_lo[tid] = ~0ull, l.part_hi[tid] = 0;
  Cut cut = {~0ull, p.k ? p.k : p.valid, p.all}, d;
  double least_y = -__builtin_inf();
  uint64_t weight[2];
  double y[2];
  int bin[2], slot[2];
  uint32_t part[2];
  __syncthreads();
  if (!l.crowded) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
      const uint32_t i = tid + j * kSampleThreads;
      slot[j] = -1;
      if (i >= n) continue;
      y[j] = sc.y(order.logit(at[j]));
      const double middle = __builtin_rint(y[j]);
      weight[j] = whole_weight(y[j] - middle);
      bin[j] = sc.bin(middle);
      slot[j] = slot_of(p, bin[j]);
      if (!p.split || slot[j] < 0) continue;
      atomicMin((unsigned long long*) &l.part_lo[slot[j]], (unsigned long long) at[j]);
      atomicMax((unsigned long long*) &l.part_hi[slot[j]], (unsigned long long) at[j]);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; j++) {
      if (slot[j] < 0) continue;
      part[j] = slot[j] << p.split;
      if (p.split) {
        const uint64_t lo = l.part_lo[slot[j]], span = l.part_hi[slot[j]] - lo;
        const int bits = span ? 64 - __builtin_clzll(span) : 0;
        part[j] += (uint32_t) ((at[j] - lo) >> (bits > p.split ? bits - p.split : 0));
      }
      atomicAdd(&l.part_n[part[j]], 1u);
      atomicAdd((unsigned long long*) &l.part_m[part[j]], (unsigned long long) weight[j]);
    }
    __syncthreads();
    // (a few's bins are its parts, and their weights are not known yet)
    const Sum own = {l.part_n[tid], small ? whole((double) l.part_m[tid] * bin_scale(tid)) : l.part_m[tid]};
    const Sum sum = scan_sum(own, l);
    l.part_m[tid] = sum.m - own.m, l.before_n[tid] = sum.n - own.n;  // before the part
    if (own.n > kCrowd) l.crowded = 1;
    if (tid == kSampleThreads - 1) l.sum = sum.m;
    __syncthreads();
  }
  if (l.crowded) {
    draw_slowly<T>(logits, a.vocab, order, p, prefix, list, l, cut, d, least_y);
  } else {
    if (small) cut.m = l.sum;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      if (slot[j] < 0) continue;
      const uint32_t i = l.before_n[part[j]] + atomicAdd(&l.filled[part[j]], 1u);
      l.sorted[i] = at[j], l.weight[i] = weight[j];
    }
    __syncthreads();
    uint32_t rank[2];
    uint64_t upto[2];
#pragma unroll
    for (int j = 0; j < 2; j++) {
      if (slot[j] < 0) continue;
      const uint32_t q = part[j], start = l.before_n[q], count = l.part_n[q], base = (uint32_t) slot[j] << p.split;
      uint32_t less = 0;
      uint64_t m = weight[j];
      for (uint32_t i = start; i < start + count; i++) {
        const bool first = l.sorted[i] < at[j];
        less += first, m += first ? l.weight[i] : 0;
      }
      rank[j] = start + less;
      const uint64_t ahead = l.part_m[q];
      upto[j] = small ? ahead + whole((double) m * bin_scale(bin[j])) : prefix.before[bin[j]] + whole((double) (m + ahead - l.part_m[base]) * bin_scale(bin[j]));
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; j++)
      if (slot[j] >= 0) l.sorted[rank[j]] = at[j], l.weight[rank[j]] = upto[j];
    __syncthreads();
    if (tid >= 64) return;
    // the first of the listed tokens that `is` holds for, as it does for all that follow
    auto first_of = [&](auto is) {
      uint32_t lo = 0, left = n;
      while (left > 1) {
        const uint32_t step = (left + 63) / 64, i = lo + tid * step + step - 1;
        const uint64_t a = __ballot(i < lo + left ? is(i) : true);
        const uint32_t s = a ? __builtin_ctzll(a) : 63;
        lo += s * step;
        left = s * step < left ? left - s * step < step ? left - s * step : step : 1;
      }
      return lo < n ? lo : n - 1;
    };
    // the i-th listed token as a cut: how many tokens of the row there are up to it
    auto cut_at = [&](uint32_t i) {
      const int b = sc.bin_of(order.logit(l.sorted[i]));
      return Cut{l.sorted[i], small ? i + 1 : prefix.ahead[b] + i - l.before_n[slot_of(p, b) << p.split] + 1, l.weight[i]};
    };
    if (p.k_bin < kBins) cut = cut_at(small ? p.k - 1 : l.before_n[slot_of(p, p.k_bin) << p.split] + p.k - prefix.ahead[p.k_bin] - 1);
    if (p.by_p) {
      const uint64_t goal = p_goal(p.part, cut.m);
      cut = cut_at(first_of([&](uint32_t i) { return l.weight[i] >= goal; }));
    }
    if (p.m_bin < kBins) {
      // the last listed token of min_p's weight or more; none of that bin: all before it
      const uint32_t i = first_of([&](uint32_t i) { return !(sc.y(order.logit(l.sorted[i])) >= p.edge); });
      const bool all = sc.y(order.logit(l.sorted[i])) >= p.edge;  // (no listed token is less)
      Cut last = {0, 0, 0};
      if (all || i) last = cut_at(all ? i : i - 1);
      if (!small && prefix.ahead[p.m_bin] > last.n) last.n = prefix.ahead[p.m_bin], last.m = prefix.before[p.m_bin];
      if (last.n < cut.n) cut.n = last.n, cut.m = last.m, least_y = p.edge;
    }
    const uint64_t goal = u_goal(p.draw, cut.m);
    d = cut_at(first_of([&](uint32_t i) { return l.weight[i] >= goal; }));
  }
  if (p.far && prefix.ahead[kBins] + p.past < cut.n) cut.n = prefix.ahead[kBins] + p.past;
  const double share = kOne / (double) cut.m;
  if (tid == 0) {
    const double z = sc.y(order.logit(d.place)), middle = __builtin_rint(z);
    a.token[t] = (int32_t) order.index(d.place);
    if (a.prob) a.prob[t] = (float) (part_weight(z - middle) * bin_scale(sc.bin(middle)) * share);
    if (a.kept) a.kept[t] = (int32_t) cut.n;
    if (a.probs) ((Drawn*) a.cuts)[t] = Drawn{cut.place, sc.by, sc.top, least_y, share};
  }
}

template <uint32_t T>
__global__ __launch_bounds__(kSampleThreads) void draw_kernel(SampleArgs a) {
  __shared__ DrawLds l;
  __shared__ Prefix prefix;
  __shared__ Plan p;
  const RowPlan* from = (const RowPlan*) a.plans + blockIdx.x;
  const uint32_t tid = threadIdx.x;
  if (tid < sizeof(Plan) / 4) ((uint32_t*) &p)[tid] = ((const uint32_t*) &from->plan)[tid];
  prefix.before[tid] = from->prefix.before[tid], prefix.ahead[tid] = from->prefix.ahead[tid];  // (what a greedy row's plan leaves is not used)
  if (tid == 0) prefix.before[kBins] = from->prefix.before[kBins], prefix.ahead[kBins] = from->prefix.ahead[kBins];
  uint64_t at[2] = {from->list[tid], from->list[tid + kSampleThreads]};  // (past the listed ones: not looked at)
  __syncthreads();
  if (p.done) return;
  const Order<T> order = {a.bits};
  draw<T>(a, blockIdx.x, order, p, prefix, from->list, at, l);
}

// a row of one slice
template <uint32_t T>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  __shared__ WholeLds l;
  const uint32_t t = blockIdx.x;
  Tokens<T, kRowPieces<T>> row = {(const uint8_t*) a.logits + t * a.stride * kv::size_of(T), 0, a.vocab};
  const Order<T> order = {a.bits};
  const Wish wish(a, t);
  uint64_t first;
  double top;
  uint32_t valid;
  scan_slice<T, false>(row, order, wish.temperature, wish.k, l.scan, first, top, valid);
  Sum bin = {0, 0};
  if (valid) bin = {l.scan.count[threadIdx.x], l.scan.mass[threadIdx.x]};
  make_plan<T>(a, t, wish, order, l, first, top, valid, bin);
  if (l.plan.done) return;
  uint32_t past = 0;
  row.loaded_between(0, l.plan, [&](float x, uint32_t i) {
    if (!planned(l.plan, x, past)) return;
    const uint32_t at = atomicAdd(&l.plan.listed, 1u);
    if (at < kList) l.list[at] = order.place(x, i);
  });
  if (past) atomicAdd(&l.plan.past, past);
  __syncthreads();
  uint64_t at[2] = {l.list[threadIdx.x], l.list[threadIdx.x + kSampleThreads]};
  draw<T>(a, t, order, l.plan, l.prefix, l.list, at, l.draw);
}

// every token's part of the kept weights
template <uint32_t T>
__global__ __launch_bounds__(kSampleThreads) void probs_kernel(SampleArgs a, uint32_t chunks) {
  __shared__ double scale[kBins];
  const uint32_t t = blockIdx.x / chunks, end = a.vocab;
  const Drawn d = ((const Drawn*) a.cuts)[t];
  const void* p = (const uint8_t*) a.logits + t * a.stride * kv::size_of(T);
  float* out = a.probs + (uint64_t) t * a.vocab;
  const Scale sc = {d.by, d.top};
  const Order<T> order = {a.bits};
  scale[threadIdx.x] = bin_scale((int) threadIdx.x) * d.share;
  __syncthreads();
  const uint32_t i = ((blockIdx.x - t * chunks) * kSampleThreads + threadIdx.x) * kPer<T>;
  if (i < end) {
    Piece<T> piece;
    piece.load(p, i, end);
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++) {
      float v = 0.0f;
      const float x = ordered<T>(piece.at(j));
      if (x > -__builtin_inff() && order.place(x, i + j) <= d.last) {
        if (d.share == 0.0) {
          v = order.place(x, i + j) == d.last ? 1.0f : 0.0f;
        } else {
          const double y = sc.y(x), middle = __builtin_rint(y);
          const int b = sc.bin(middle);
          if (b < kBins && y >= d.least_y) v = (float) (part_weight(y - middle) * scale[b]);
        }
      }
      if (i + j < end) out[i + j] = v;
    }
  }
}

inline int index_bits(uint32_t vocab) { return vocab > 1 ? 32 - __builtin_clz(vocab - 1) : 0; }
// a row of up to 32768 tokens is one slice. VALUES: bf16's tokens are counted by value, where there are many: a slice then costs the same
// whatever it holds (its values are put into bins at the end), so it is as long as leaves 512 of them. 256 / 128 / 64 / 1 rows of
// 129024: 60 / 44 / 35 / 29 us by values, 76 / 49 / 37 / 28 token by token
constexpr uint32_t kRow = 32768;
inline bool by_values(const OsmosSample* a) {
  return a->type == OSMOS_BF16 && a->vocab > kRow && (uint64_t) a->n * ((a->vocab + kValueSlice - 1) / kValueSlice) >= 512;
}
inline uint32_t slice_of(const OsmosSample* a) {
  if (a->vocab <= kRow) return kRow;
  if (!by_values(a)) return kSlice;
  const uint32_t rounds = (a->vocab + kValueSlice - 1) / kValueSlice;
  const uint64_t each = (uint64_t) a->n * rounds / 512;
  return kValueSlice * (uint32_t) (each < 1 ? 1 : each < rounds ? each : rounds);
}
inline uint32_t slices_of(const OsmosSample* a) { return (a->vocab + slice_of(a) - 1) / slice_of(a); }
inline uint64_t round256(uint64_t n) { return (n + 255) / 256 * 256; }
struct SampleRoom {
  uint64_t parts, plans, cuts;
};
inline SampleRoom room_of(const OsmosSample* a) {
  const uint64_t rows = a->n, slices = slices_of(a);
  return {a->vocab > kRow ? round256(rows * slices * sizeof(Part)) : 0, a->vocab > kRow ? round256(rows * sizeof(RowPlan)) : 0,
          a->probs ? round256(rows * sizeof(Drawn)) : 0};
}

template <uint32_t T, bool VALUES>
bool sample_launch(const SampleArgs& a, hipStream_t s) {
  constexpr uint32_t list_each = kListThreads * kPer<T> * kListPieces, probs_each = kSampleThreads * kPer<T>;
  const uint64_t blocks = (a.vocab + list_each - 1) / list_each, chunks = (a.vocab + probs_each - 1) / probs_each;
  if (!launches((uint64_t) a.n * a.slices, kSampleThreads) || !launches(a.n * blocks, kListThreads) ||
      (a.probs && !launches(a.n * chunks, kSampleThreads)))
    return false;
  if (a.vocab > kRow) {
    scan_kernel<T, VALUES><<<a.n * a.slices, kSampleThreads, 0, s>>>(a);
    plan_kernel<T><<<a.n, kSampleThreads, 0, s>>>(a);
    list_kernel<T><<<(uint32_t) (a.n * blocks), kListThreads, 0, s>>>(a, (uint32_t) blocks);
    draw_kernel<T><<<a.n, kSampleThreads, 0, s>>>(a);
  } else {
    sample_kernel<T><<<a.n, kSampleThreads, 0, s>>>(a);
  }
  if (a.probs) probs_kernel<T><<<(uint32_t) (a.n * chunks), kSampleThreads, 0, s>>>(a, (uint32_t) chunks);
  return hipGetLastError() == hipSuccess;
}

}  // namespace rows
}  // namespace osm

using namespace osm;

extern "C" OSM_API uint64_t osmos_sample_workspace(const OsmosSample* a) {
  if (!rows::sample_ok(a)) return 0;
  const rows::SampleRoom r = rows::room_of(a);
  return r.parts + r.plans + r.cuts;
}

extern "C" OSM_API bool osmos_sample(const OsmosSample* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  const uint64_t need = osmos_sample_workspace(a);
  if (!rows::sample_ok(a) || (need && (!workspace || !rows::aligned(workspace, 256) || workspace_bytes < need))) return false;
  const rows::SampleRoom r = rows::room_of(a);
  uint8_t* w = (uint8_t*) workspace;
  const rows::SampleArgs b = {a->logits, a->u, a->temperature, a->top_p, a->min_p, a->top_k, a->token, a->kept, a->prob, a->probs, a->stride,
                              a->n, a->vocab, rows::slices_of(a), rows::slice_of(a), rows::index_bits(a->vocab), w, w + r.parts,
                              w + r.parts + r.plans};
  const hipStream_t on = (hipStream_t) stream;
  return a->type == OSMOS_F32 ? rows::sample_launch<OSMOS_F32, false>(b, on)
         : a->type == OSMOS_F16 ? rows::sample_launch<OSMOS_F16, false>(b, on)
         : rows::by_values(a) ? rows::sample_launch<OSMOS_BF16, true>(b, on) : rows::sample_launch<OSMOS_BF16, false>(b, on);
}
