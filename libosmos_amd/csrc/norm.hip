// libosmos MI355X - osmos_norm (include/osmos_rows.h): the residual's addition, the root-mean-square norm and the forms that the
// products read, in one pass over the rows.
#include "rowshost.h"
#include "lanes.h"
#include "x16.h"

namespace osm {
namespace rows {

// 16 bytes of values as floats, at any address that their type allows
template <uint32_t T> constexpr int per() { return T == OSMOS_F32 ? 4 : 8; }
typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));
template <int N> struct Halves {
  typedef _Float16 F __attribute__((ext_vector_type(N), aligned(2)));
  typedef __bf16 B __attribute__((ext_vector_type(N), aligned(2)));
};

template <int N>
__device__ inline void load(uint32_t type, const void* p, uint64_t at, float* x) {
  if (type == OSMOS_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4_u v = gload<f32x4_u>((const float*) p + at + i);
      x[i] = v[0], x[i + 1] = v[1], x[i + 2] = v[2], x[i + 3] = v[3];
    }
  } else if (type == OSMOS_F16) {
    const typename Halves<N>::F v = gload<typename Halves<N>::F>((const _Float16*) p + at);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = (float) v[i];
  } else {
    const typename Halves<N>::B v = gload<typename Halves<N>::B>((const __bf16*) p + at);
#pragma unroll
    for (int i = 0; i < N; i++) x[i] = (float) v[i];
  }
}
template <int N>
__device__ inline void store(uint32_t type, void* p, uint64_t at, const float* x) {
  if (type == OSMOS_F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *(f32x4_u*) ((float*) p + at + i) = f32x4_u{x[i], x[i + 1], x[i + 2], x[i + 3]};
  } else if (type == OSMOS_F16) {
    typename Halves<N>::F v;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = (_Float16) x[i];
    *(typename Halves<N>::F*) ((_Float16*) p + at) = v;
  } else {
    typename Halves<N>::B v;
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = (__bf16) x[i];
    *(typename Halves<N>::B*) ((__bf16*) p + at) = v;
  }
}
__device__ inline void store1(uint32_t type, void* p, uint64_t at, float x) {
  if (type == OSMOS_F32) ((float*) p)[at] = x;
  else if (type == OSMOS_F16) ((_Float16*) p)[at] = (_Float16) x;
  else ((__bf16*) p)[at] = (__bf16) x;
}
// the first `left` of N values (all of them but in a row's last, partial piece: TAIL, whether rows have one)
template <int N, bool TAIL>
__device__ inline void load_part(uint32_t type, const void* p, uint64_t at, uint32_t left, float* x) {
  if (!TAIL || left >= N) return load<N>(type, p, at, x);
  uint32_t w[N];  // (all of them on their way together: one after the other 700 rows of 4999 take 8.9 us, so 7.5)
  if (type == OSMOS_F32) {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = gload<uint32_t>((const uint32_t*) p + at + ((uint32_t) i < left ? i : 0));
  } else {
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = gload<uint16_t>((const uint16_t*) p + at + ((uint32_t) i < left ? i : 0));
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float v = type == OSMOS_F32 ? __uint_as_float(w[i]) : type == OSMOS_F16 ? __half2float(__ushort_as_half((unsigned short) w[i])) : __uint_as_float(w[i] << 16);
    x[i] = (uint32_t) i < left ? v : 0.0f;
  }
}
template <int N, bool TAIL>
__device__ inline void store_part(uint32_t type, void* p, uint64_t at, uint32_t left, const float* x) {
  if (!TAIL || left >= N) return store<N>(type, p, at, x);
#pragma unroll
  for (int i = 0; i < N; i++)
    if ((uint32_t) i < left) store1(type, p, at + i, x[i]);
}

// 1 / sqrt(a) for a >= 0, within a few units of float64: the hardware's estimate (2^-26 or better) and two of Newton's steps
__device__ inline double rsqrt64(double a) {
  const double e = __builtin_amdgcn_rsq(a);
  double y = e;
#pragma unroll
  for (int i = 0; i < 2; i++) y = __builtin_fma(y * 0.5, __builtin_fma(-a * y, y, 1.0), y);
  return a > 0.0 && a < __builtin_inf() ? y : e;
}

struct NormArgs {
  const void *x, *add;  // (sum may be either: no restrict)
  void* sum;
  const void* weight;
  void* out;
  _Float16* x16;
  int32_t* overflow;
  int8_t* codes;
  float* scales;
  uint64_t x_stride, add_stride, sum_stride, out_stride;
  uint32_t weight_type, out_type, n, dim;
  float eps, offset;
  double part;      // 1 / dim
  uint32_t waves;   // a row's; 1: each wave of the workgroup a row of its own
  bool tiles;
};

// a row a workgroup (short ones: a wave), its values in registers between the sum of their squares and their stores: K pieces of 16
// bytes a thread. bound by memory where the rows are many: 4096 rows of 6144 floats and as many to add, the sums and f16 tiles
// written, 69 us for 352 MB (5.1 TB/s, more than a large copy reaches); by latency where they are few: one row of 4096 3.0 us, the launch,
// one trip to memory, the sum over the row (lane moves, then LDS) and the stores
template <uint32_t T, int K, bool TAIL>
__global__ __launch_bounds__(1024) void norm_kernel(NormArgs a) {
  constexpr int N = per<T>();
  __shared__ double sums[16];
  const uint32_t lanes = a.waves * 64, wave = threadIdx.x / 64;
  uint32_t t = a.waves > 1 ? blockIdx.x : blockIdx.x * (blockDim.x / 64) + wave;
  // workgroups go to the 8 XCDs in turn: the 16 rows of a tile, whose values lie in the same lines, to one of them (4096 rows of
  // 6144 floats 96 -> 80 us: a line is written back once, not in parts by several)
  if (a.tiles && a.waves > 1 && blockIdx.x < gridDim.x / 128 * 128) t = blockIdx.x / 128 * 128 + blockIdx.x % 8 * 16 + blockIdx.x / 8 % 16;
  const uint32_t at = a.waves > 1 ? threadIdx.x : threadIdx.x & 63;
  const uint32_t pieces = (a.dim + N - 1) / N;
  const bool live = t < a.n;  // (a row past the last: of a tile's rest, or none)
  float s[K][N];
  double ss = 0.0;
  if (live) {
#pragma unroll
    for (int k = 0; k < K; k++) {
      const uint32_t c = at + k * lanes;
      if (c < pieces) load_part<N, TAIL>(T, a.x, t * a.x_stride + c * N, a.dim - c * N, s[k]);
      else
#pragma unroll
        for (int i = 0; i < N; i++) s[k][i] = 0.0f;
    }
    if (a.add)
#pragma unroll
      for (int k = 0; k < K; k++) {
        const uint32_t c = at + k * lanes;
        float d[N];
        if (c < pieces) {
          load_part<N, TAIL>(T, a.add, t * a.add_stride + c * N, a.dim - c * N, d);
#pragma unroll
          for (int i = 0; i < N; i++) s[k][i] = __fadd_rn(s[k][i], d[i]);
        }
      }
#pragma unroll
    for (int k = 0; k < K; k++) {
      const uint32_t c = at + k * lanes;
      if (a.sum && c < pieces) store_part<N, TAIL>(T, a.sum, t * a.sum_stride + c * N, a.dim - c * N, s[k]);
#pragma unroll
      for (int i = 0; i < N; i++) ss = __builtin_fma((double) s[k][i], (double) s[k][i], ss);
    }
  }
  if (!a.out && !a.x16 && !a.codes) return;
  // (the weights are on their way meanwhile, where there is room for them)
  constexpr bool early = K * N <= 16;
  float w[early ? K : 1][N];
  if constexpr (early)
    if (a.weight && live)
#pragma unroll
      for (int k = 0; k < K; k++) {
        const uint32_t c = at + k * lanes;
        if (c < pieces) load_part<N, TAIL>(a.weight_type, a.weight, c * N, a.dim - c * N, w[k]);
      }
  ss = wave_total(ss);
  if (a.waves > 1) {
    if (at % 64 == 0) sums[wave] = ss;
    __syncthreads();
    ss = 0.0;
    for (uint32_t w = 0; w < a.waves; w++) ss += sums[w];
  }
  const float r = (float) rsqrt64(__builtin_fma(ss, a.part, (double) a.eps));
  bool over = false;
#pragma unroll
  for (int k = 0; k < K; k++) {
    const uint32_t c = at + k * lanes;
    if (c >= pieces) break;
    float y[N];
    if (!live) {
      if (!a.x16 || t >= (a.n + 15) / 16 * 16) break;
#pragma unroll
      for (int i = 0; i < N; i++) y[i] = 0.0f;
    } else {
      float(&own)[N] = w[early ? k : 0];
      if constexpr (!early)
        if (a.weight) load_part<N, TAIL>(a.weight_type, a.weight, c * N, a.dim - c * N, own);
#pragma unroll
      for (int i = 0; i < N; i++)
        y[i] = a.weight ? __fmul_rn(__fmul_rn(s[k][i], r), __fadd_rn(own[i], a.offset))
                        : __fmul_rn(__fmul_rn(s[k][i], r), __fadd_rn(1.0f, a.offset));
      if (a.out) store_part<N, TAIL>(a.out_type, a.out, t * a.out_stride + c * N, a.dim - c * N, y);
      if (a.codes) {
        float am = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) am = fmaxf(am, fabsf(y[i]));
        am = fmaxf(am, xor_lane(am, 1));
        am = fmaxf(am, xor_lane(am, 2));
        if (N == 4) am = fmaxf(am, xor_lane(am, 4));
        const float inv = am > 0.0f ? __fdiv_rn(127.0f, am) : 0.0f;
        uint32_t* q = (uint32_t*) (a.codes + (uint64_t) t * a.dim + c * N);
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          uint32_t v = 0;
#pragma unroll
          for (int j = 0; j < 4; j++) v |= ((uint32_t) (int) rintf(__fmul_rn(y[i + j], inv)) & 0xFF) << (8 * j);
          q[i / 4] = v;
        }
        if (c % (32 / N) == 0) a.scales[(uint64_t) t * (a.dim / 32) + c / (32 / N)] = __fdiv_rn(am, 127.0f);
      }
    }
    if (a.x16) {
      _Float16 h[N];
#pragma unroll
      for (int i = 0; i < N; i++) h[i] = x16_round(y[i], over);
      __builtin_memcpy(__builtin_assume_aligned(a.x16 + x16_at(t, c * N, a.dim), 2 * N), h, 2 * N);
    }
  }
  if (over) *a.overflow = 1;
}

template <uint32_t T, bool TAIL>
auto norm_of(uint32_t k) {
  return k <= 1 ? norm_kernel<T, 1, TAIL> : k <= 2 ? norm_kernel<T, 2, TAIL> : k <= 4 ? norm_kernel<T, 4, TAIL>
         : k <= 8 ? norm_kernel<T, 8, TAIL> : norm_kernel<T, 64 / per<T>(), TAIL>;
}

template <uint32_t T>
bool norm_launch(const OsmosNorm* a, hipStream_t s) {
  const uint32_t pieces = (a->dim + per<T>() - 1) / per<T>(), rows = a->x16 ? (a->n + 15) / 16 * 16 : a->n;
  NormArgs b = {a->x, a->add, a->sum, a->weight, a->out, (_Float16*) a->x16, a->overflow, a->codes, a->scales, a->x_stride, a->add_stride,
                a->sum_stride, a->out_stride, a->weight_type, a->out_type, a->n, a->dim, a->eps, a->offset, 1.0 / a->dim, 0, a->x16 != nullptr};
  // as many waves as there are pieces for, 16 at most (then 2 pieces a thread and more). for such waves (a half, a quarter, an eighth of
  // them, 16 at most), sums written too: one row of 4096 floats into tiles 3.7 us (3.6, 4.4, 6.9), 48 of 2048 3.5 (3.8, 4.7, 7.4), 1000
  // of 4096 12.7 (10.5, 11.2, 13.9), 4096 of 6144 68.5 (68.8, 72.9, 83.0), 8192 bf16 rows of 4096 into rows 39.7 (41.7, 43.2, 46.0): the
  // best, or 3 % from it, but for the 1000 rows
  const uint32_t waves = (pieces + 63) / 64;
  b.waves = waves > 16 ? 16 : waves;
  const uint32_t k = (pieces + b.waves * 64 - 1) / (b.waves * 64);
  if (!launches(b.waves > 1 ? rows : (rows + 3) / 4, b.waves > 1 ? b.waves * 64 : 256)) return false;
  auto* kernel = a->dim % per<T>() ? norm_of<T, true>(k) : norm_of<T, false>(k);
  if (b.waves > 1) kernel<<<rows, b.waves * 64, 0, s>>>(b);
  else kernel<<<(rows + 3) / 4, 256, 0, s>>>(b);
  return hipGetLastError() == hipSuccess;
}

}  // namespace rows
}  // namespace osm

using namespace osm;

extern "C" OSM_API bool osmos_norm(const OsmosNorm* a, void* stream) {
  if (!rows::norm_ok(a)) return false;
  return a->type == OSMOS_F32 ? rows::norm_launch<OSMOS_F32>(a, (hipStream_t) stream)
         : a->type == OSMOS_F16 ? rows::norm_launch<OSMOS_F16>(a, (hipStream_t) stream) : rows::norm_launch<OSMOS_BF16>(a, (hipStream_t) stream);
}
