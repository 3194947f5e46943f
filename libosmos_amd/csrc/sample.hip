// libosmos MI355X - osmos_sample (include/osmos_rows.h): one token for each row of logits.
//
// tokens are put into bins of their logits, 23 an octave of weight: y = logit x 23 log2(e) / T, bin floor(y), its weight
// 2^(y / 23). a bin's weights are summed as whole numbers of 2^-42 of its lower edge's weight, so that the sums do not depend on
// their order; a prefix of the tokens' order is whole bins and then some of one bin's tokens, which are found by their logits'
// bits and indexes, 1024 parts of what is left at a time.
#include "rowshost.h"
#include "common.h"

namespace osm {
namespace rows {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBins = 1024;           // 44.5 octaves below the greatest weight: what is further down is in no bin
constexpr double kOctave = 23.0;
constexpr double kOne = 4398046511104.0;  // 2^42: 2^20 tokens of up to 2^(1 / 23) stay under 2^63

// a logit as the order takes it
template <uint32_t T>
__device__ inline float logit_at(const void* p, uint64_t i) {
  float x;
  if constexpr (T == OSMOS_F32) x = gload<float>((const float*) p + i);
  else if constexpr (T == OSMOS_F16) x = (float) gload<_Float16>((const _Float16*) p + i);
  else x = (float) gload<__bf16>((const __bf16*) p + i);
  return x != x ? -__builtin_inff() : fminf(x, 3.402823466e38f);
}
// (the greatest first, the lower index first among equals)
__device__ inline uint64_t place(float x, uint32_t i) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // (-0 is 0)
  return (uint64_t) (b & 0x80000000u ? b : ~b & 0x7FFFFFFFu) << 32 | i;
}

// 2^(f / 23) for 0 <= f < 1, within 2^-47
__device__ inline double part_weight(double f) {
  const double x = f * (0.69314718055994530942 / kOctave);
  double r = __builtin_fma(x, 1.0 / 720, 1.0 / 120);
  r = __builtin_fma(x, r, 1.0 / 24);
  r = __builtin_fma(x, r, 1.0 / 6);
  r = __builtin_fma(x, r, 0.5);
  r = __builtin_fma(x, r, 1.0);
  return __builtin_fma(x, r, 1.0);
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
};

struct Sum {
  uint32_t n;  // tokens
  uint64_t m;  // their weights
};

struct SampleLds {
  uint32_t count[kBins];
  uint64_t mass[kBins];
  uint64_t before[kBins + 1];  // the bins' prefix sums, of kOne the greatest bin's edge
  uint32_t ahead[kBins + 1];
  double scale[kBins];         // a bin's weight by the first's
  uint32_t part_n[kBins];
  uint64_t part_m[kBins];
  Sum wave[kSampleWaves];
  uint64_t word[kSampleWaves], found[4];
};

__device__ inline uint64_t shfl64(uint64_t v, int lane) {
  return (uint64_t) (uint32_t) __shfl((int) (v >> 32), lane) << 32 | (uint32_t) __shfl((int) v, lane);
}
// inclusive sums over the workgroup's threads in their order
__device__ inline Sum scan_sum(Sum x, SampleLds& l) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x / 64;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t n = (uint32_t) __shfl_up((int) x.n, o);
    const uint64_t m = (uint64_t) (uint32_t) __shfl_up((int) (x.m >> 32), o) << 32 | (uint32_t) __shfl_up((int) x.m, o);
    if (lane >= o) x.n += n, x.m += m;
  }
  __syncthreads();
  if (lane == 63) l.wave[wave] = x;
  __syncthreads();
  for (int w = 0; w < wave; w++) x.n += l.wave[w].n, x.m += l.wave[w].m;
  return x;
}
__device__ inline uint64_t least(uint64_t x, SampleLds& l) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const uint64_t y = shfl64(x, (threadIdx.x & 63) ^ o);
    x = y < x ? y : x;
  }
  __syncthreads();
  if (threadIdx.x % 64 == 0) l.word[threadIdx.x / 64] = x;
  __syncthreads();
  x = l.word[0];
  for (int w = 1; w < kSampleWaves; w++) x = l.word[w] < x ? l.word[w] : x;
  return x;
}

// where a row's logits lie on the bins' scale
struct Scale {
  double by, top;  // bins a unit of logit; the first bin's floor
  __device__ inline double y(float x) const { return (double) x * by; }
  __device__ inline int bin(double floor) const {  // kBins: none
    const double b = top - floor;
    return b < kBins ? (int) b : kBins;
  }
};

struct Cut {
  uint64_t place;  // the last token
  uint32_t n;      // how many tokens up to it
  uint64_t m;      // their weights
};

template <uint32_t T>
struct Row {
  const void* p;
  uint32_t vocab;
  template <typename F>
  __device__ inline void each(F f) const {
    for (uint32_t i = threadIdx.x; i < vocab; i += kSampleThreads) {
      const float x = logit_at<T>(p, i);
      if (x > -__builtin_inff()) f(x, i);
    }
  }
};

// the first token of bin b with at least `rank` tokens of the bin up to it (MASS: with at least `goal` of weight up to it)
template <bool MASS, typename R>
__device__ Cut find(const R& row, const Scale& sc, SampleLds& l, int b, uint32_t rank, uint64_t goal) {
  const double scale = l.scale[b];
  const uint64_t before = l.before[b];
  uint64_t lo = ~0ull, hi = ~0ull;  // (hi: the greatest place, inverted)
  row.each([&](float x, uint32_t i) {
    if (sc.bin(__builtin_floor(sc.y(x))) != b) return;
    const uint64_t at = place(x, i);
    lo = at < lo ? at : lo, hi = ~at < hi ? ~at : hi;
  });
  lo = least(lo, l), hi = ~least(hi, l);
  Sum base = {0, 0};
  for (;;) {
    const int bits = hi > lo ? 64 - __builtin_clzll(hi - lo) : 0, shift = bits > 10 ? bits - 10 : 0;
    __syncthreads();
    l.part_n[threadIdx.x] = 0, l.part_m[threadIdx.x] = 0;
    __syncthreads();
    row.each([&](float x, uint32_t i) {
      const double y = sc.y(x), floor = __builtin_floor(y);
      if (sc.bin(floor) != b) return;
      const uint64_t at = place(x, i);
      if (at < lo || at > hi) return;
      atomicAdd(&l.part_n[(at - lo) >> shift], 1u);
      atomicAdd((unsigned long long*) &l.part_m[(at - lo) >> shift], (unsigned long long) whole(part_weight(y - floor) * kOne));
    });
    __syncthreads();
    const Sum own = {l.part_n[threadIdx.x], l.part_m[threadIdx.x]};
    Sum sum = scan_sum(own, l);
    sum.n += base.n, sum.m += base.m;
    const Sum past = {sum.n - own.n, sum.m - own.m};
    const bool here = MASS ? before + whole((double) sum.m * scale) >= goal && before + whole((double) past.m * scale) < goal
                           : sum.n >= rank && past.n < rank;
    if (here) l.found[0] = threadIdx.x, l.found[1] = shift ? past.n : sum.n, l.found[2] = shift ? past.m : sum.m;
    __syncthreads();
    base.n = (uint32_t) l.found[1], base.m = l.found[2];
    lo += l.found[0] << shift;
    if (!shift) return Cut{lo, l.ahead[b] + base.n, before + whole((double) base.m * scale)};
    const uint64_t last = lo + (1ull << shift) - 1;
    hi = last < hi ? last : hi;
  }
}

template <uint32_t T>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs a) {
  __shared__ SampleLds l;
  const uint32_t t = blockIdx.x, tid = threadIdx.x;
  const Row<T> row = {(const uint8_t*) a.logits + t * a.stride * kv::size_of(T), a.vocab};
  const float temperature = a.temperature ? a.temperature[t] : 1.0f;
  uint64_t first = ~0ull;
  row.each([&](float x, uint32_t i) {
    const uint64_t at = place(x, i);
    first = at < first ? at : first;
  });
  first = least(first, l);
  float* probs = a.probs ? a.probs + (uint64_t) t * a.vocab : nullptr;
  const bool greedy = !(temperature > 0.0f);
  if (first == ~0ull || greedy) {
    const bool none = first == ~0ull;
    if (tid == 0) {
      a.token[t] = none ? -1 : (int32_t) (uint32_t) first;
      if (a.prob) a.prob[t] = none ? 0.0f : 1.0f;
      if (a.kept) a.kept[t] = none ? 0 : 1;
    }
    if (probs)
      for (uint32_t i = tid; i < a.vocab; i += kSampleThreads) probs[i] = !none && i == (uint32_t) first ? 1.0f : 0.0f;
    return;
  }
  const float most = logit_at<T>(row.p, (uint32_t) first);
  Scale sc;
  sc.by = kOctave * 1.4426950408889634074 / (double) temperature;
  sc.top = __builtin_floor(sc.y(most));
  l.count[tid] = 0, l.mass[tid] = 0;
  if (tid < 4) l.found[tid] = 0;
  l.scale[tid] = exp2(-(double) (int) tid / kOctave);
  __syncthreads();
  uint32_t valid = 0;
  row.each([&](float x, uint32_t i) {
    const double y = sc.y(x), floor = __builtin_floor(y);
    const int b = sc.bin(floor);
    valid++;
    if (b >= kBins) return;
    atomicAdd(&l.count[b], 1u);
    atomicAdd((unsigned long long*) &l.mass[b], (unsigned long long) whole(part_weight(y - floor) * kOne));
  });
  {
    const Sum all = scan_sum(Sum{valid, 0}, l);
    if (tid == kSampleThreads - 1) l.found[0] = all.n;
    __syncthreads();
    valid = (uint32_t) l.found[0];
    const Sum sum = scan_sum(Sum{l.count[tid], whole((double) l.mass[tid] * l.scale[tid])}, l);
    l.ahead[tid + 1] = sum.n, l.before[tid + 1] = sum.m;
    if (tid == 0) l.ahead[0] = 0, l.before[0] = 0;
    __syncthreads();
  }
  Cut cut = {~0ull, valid, l.before[kBins]};
  auto by_rank = [&](uint32_t rank) {
    if (rank > l.ahead[kBins]) {  // (among tokens of no weight)
      cut.n = rank;
      return;
    }
    if (l.ahead[tid + 1] >= rank && l.ahead[tid] < rank) l.found[3] = tid;
    __syncthreads();
    const int b = (int) l.found[3];
    cut = find<false>(row, sc, l, b, rank - l.ahead[b], 0);
    __syncthreads();
  };
  auto by_mass = [&](uint64_t goal) {
    if (l.before[tid + 1] >= goal && l.before[tid] < goal) l.found[3] = tid;
    __syncthreads();
    const int b = (int) l.found[3];
    const Cut c = find<true>(row, sc, l, b, 0, goal);
    __syncthreads();
    return c;
  };
  const int32_t k = a.top_k ? a.top_k[t] : 0;
  if (k > 0 && (uint32_t) k < cut.n) by_rank((uint32_t) k);
  const float p = a.top_p ? a.top_p[t] : 1.0f;
  if (p < 1.0f) {
    const double goal = (double) cut.m * (double) (p > 0.0f ? p : 0.0f);
    cut = by_mass(goal > 1.0 ? (uint64_t) __builtin_ceil(goal) : 1);
  }
  const float min_p = a.min_p ? a.min_p[t] : 0.0f;
  if (min_p > 0.0f) {
    const double edge = sc.y(most) + kOctave * log2((double) (min_p < 1.0f ? min_p : 1.0f));
    const int b = sc.bin(__builtin_floor(edge));
    if (b < kBins) {
      uint32_t in = 0;
      row.each([&](float x, uint32_t i) {
        const double y = sc.y(x);
        in += y >= edge && sc.bin(__builtin_floor(y)) == b;
      });
      const Sum all = scan_sum(Sum{in, 0}, l);
      if (tid == kSampleThreads - 1) l.found[0] = all.n;
      __syncthreads();
      const uint32_t n = l.ahead[b] + (uint32_t) l.found[0];
      __syncthreads();
      if (n < cut.n) by_rank(n ? n : 1);
    }
  }
  const float u = a.u[t];
  uint64_t goal = (uint64_t) __builtin_floor((double) cut.m * (double) (u > 0.0f ? u < 1.0f ? u : 0.99999994f : 0.0f)) + 1;
  if (goal > cut.m) goal = cut.m;
  const Cut drawn = by_mass(goal);
  const uint32_t token = (uint32_t) drawn.place;
  const double by = 1.0 / ((double) cut.m / kOne);
  auto share = [&](float x) {
    const double y = sc.y(x), floor = __builtin_floor(y);
    const int b = sc.bin(floor);
    return b < kBins ? (float) (part_weight(y - floor) * l.scale[b] * by) : 0.0f;
  };
  if (tid == 0) {
    a.token[t] = (int32_t) token;
    if (a.prob) a.prob[t] = share(logit_at<T>(row.p, token));
    if (a.kept) a.kept[t] = (int32_t) cut.n;
  }
  if (probs)
    for (uint32_t i = tid; i < a.vocab; i += kSampleThreads) {
      const float x = logit_at<T>(row.p, i);
      probs[i] = x > -__builtin_inff() && place(x, i) <= cut.place ? share(x) : 0.0f;
    }
}

}  // namespace rows
}  // namespace osm

using namespace osm;

extern "C" OSM_API uint64_t osmos_sample_workspace(const OsmosSample* a) { return 0; }

extern "C" OSM_API bool osmos_sample(const OsmosSample* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  if (!rows::sample_ok(a)) return false;
  const rows::SampleArgs b = {a->logits, a->u, a->temperature, a->top_p, a->min_p, a->top_k, a->token, a->kept, a->prob, a->probs, a->stride,
                              a->n, a->vocab};
  auto* kernel = a->type == OSMOS_F32 ? rows::sample_kernel<OSMOS_F32> : a->type == OSMOS_F16 ? rows::sample_kernel<OSMOS_F16> : rows::sample_kernel<OSMOS_BF16>;
  kernel<<<a->n, rows::kSampleThreads, 0, (hipStream_t) stream>>>(b);
  return hipGetLastError() == hipSuccess;
}
