// libosmos MI355X - osmos_rope, osmos_rope_append, osmos_rope_turns (include/osmos_rows.h): heads normed and turned to their
// positions, on packed rows or on their way into the paged cache.
#include "rowshost.h"
#include "kvcache.h"

namespace osm {
namespace rows {

// sine and cosine of pos x turn turns: the product exactly (what its rounding leaves is added to its fraction: at position 2^31 the
// rounding alone is up to 2^-25 of a turn, more than the angle's own to float), the fraction of a quarter turn in float64, then the
// series on [-pi/4, pi/4] in float (the first terms left out are under 2^-28.5 of the results')
__device__ inline void sin_cos(double pos, double turn, float& s, float& c) {
  const double t = pos * turn, q = 4.0 * (t - __builtin_rint(t) + __builtin_fma(pos, turn, -t)), k = __builtin_rint(q);
  const float x = (float) ((q - k) * 1.5707963267948966), z = x * x;
  float a = __builtin_fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  a = __builtin_fmaf(z, a, 8.3333333e-3f);
  a = __builtin_fmaf(z, a, -0.16666667f);
  a = __builtin_fmaf(z * x, a, x);
  float b = __builtin_fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  b = __builtin_fmaf(z, b, -1.3888889e-3f);
  b = __builtin_fmaf(z, b, 4.1666668e-2f);
  b = __builtin_fmaf(z, b, -0.5f);
  b = __builtin_fmaf(z, b, 1.0f);
  const int n = (int) k;  // (-4 .. 4 where the turns are under 2^53)
  s = n & 1 ? b : a, c = n & 1 ? a : b;
  s = n & 2 ? -s : s, c = (n + 1) & 2 ? -c : c;
}

struct RopeArgs {
  const double* turns;
  const float *q_weight, *k_weight;
  const uint8_t *q, *k, *v;
  uint8_t *q_out, *k_out;
  uint64_t q_stride, q_head, k_stride, k_head, v_stride, v_head, q_out_stride, q_out_head, k_out_stride, k_out_head;
  uint32_t out_type, heads, kv_heads, n, dim, rot, layout;
  float scale, eps, offset;
  uint32_t group;       // lanes a head: dim / 8 up to a power of two
  uint32_t parts;       // waves a row
};
struct Pages {
  uint8_t* data;
  const float* scale;
  uint32_t pages, page;
  uint64_t plane;
};

__device__ inline void store8_as(uint32_t type, void* p, const float (&x)[8]) {
  if (type == OSMOS_F32) kv::store8<OSMOS_F32>(p, x);
  else if (type == OSMOS_F16) kv::store8<OSMOS_F16>(p, x);
  else kv::store8<OSMOS_BF16>(p, x);
}

// a wave's LDS writes before its reads that follow (the wave's own: it does not wait for others)
__device__ inline void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

constexpr int kRopeWaves = 4;

// a wave takes a row, or a part of its heads: `group` lanes a head, 8 values a lane, so that a lane has the same values of all its
// heads. the wave makes each of the row's angles once, a lane one or two, and hands them round by LDS (each lane its own eight: 700
// rows 12.1 us, so 10.1). bound by memory for many rows (8192 bf16 rows of 40 heads of 128: 37 us for 168 MB, 4.5 TB/s), by the chain
// of launch, lengths, table and stores for few (one row 4.0 us in all, 64 rows normed into 8 bits 6.7); kAhead: heads it holds the loads of. a half layout's other values come from the other lane by LDS
template <uint32_t IN, uint32_t DST, int kAhead>
__global__ __launch_bounds__(64 * kRopeWaves) void rope_kernel(RopeArgs a, const int32_t* __restrict__ positions, kv::Step st, Pages pg) {
  __shared__ float lds[kRopeWaves][64 * 8];
  __shared__ float2 angle[kRopeWaves][OSMOS_ATTN_MAX_DIM / 2];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const uint32_t unit = blockIdx.x * kRopeWaves + wave, t = unit / a.parts, part = unit - t * a.parts;
  if (t >= a.n) return;
  const uint32_t g = lane & (a.group - 1), first = lane / a.group, each = 64 / a.group;
  const uint32_t turned = a.heads + a.kv_heads, all = turned + (DST ? a.kv_heads : 0);
  const bool active = g * 8 < a.dim;
  float x[kAhead][8], scale[kAhead];
  auto load = [&](uint32_t h0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
      const uint32_t h = h0 + i * each * a.parts;
      if (h >= all || !active) {
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = 0.0f;
        continue;
      }
      if (DST == OSMOS_F8 && pg.scale && h >= a.heads) scale[i] = pg.scale[h - a.heads];  // (keys', then values')
      const uint8_t* p = h < a.heads ? a.q + (t * a.q_stride + h * a.q_head) * kv::size_of(IN)
                         : h < turned ? a.k + (t * a.k_stride + (h - a.heads) * a.k_head) * kv::size_of(IN)
                                      : a.v + (t * a.v_stride + (h - turned) * a.v_head) * kv::size_of(IN);
      kv::load8<IN>(p + g * 8 * kv::size_of(IN), x[i]);
    }
  };
  uint32_t h0 = part * each + first;
  load(h0);
  // (what does not hang on the position is on its way while that is looked up)
  const uint32_t half = a.rot / 2;
  const bool pairs = a.layout == OSMOS_ROPE_PAIRS;
  const uint32_t mine = g * 8 >= a.rot ? 0 : a.rot - g * 8;  // the lane's first values that turn
  double turns[2];  // (a lane's angles: pairs lane and lane + 64)
#pragma unroll
  for (int i = 0; i < 2; i++) turns[i] = lane + 64 * i < half ? a.turns[lane + 64 * i] : 0.0;
  float wq[8], wk[8];
  if (a.q_weight || a.k_weight)
#pragma unroll
    for (int j = 0; j < 8; j++) {
      wq[j] = a.q_weight && active ? __fadd_rn(a.q_weight[g * 8 + j], a.offset) : 1.0f;
      wk[j] = a.k_weight && active ? __fadd_rn(a.k_weight[g * 8 + j], a.offset) : 1.0f;
    }
  int pos;
  uint32_t id = 0;  // (the row's page)
  if constexpr (DST != 0) {
    kv::Seq q;
    if (!kv::sequence_of(st, (int) t, pg.page, q)) return;
    pos = q.len - (q.row0 + q.rows - (int) t);
    if ((int) t < q.row0 || (int) t >= q.row0 + q.rows || pos < 0 || pos >= q.end) return;
    id = (uint32_t) gload<int>(q.table + (uint32_t) pos / pg.page);
  } else {
    pos = positions[t];
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (64 * i < (int) half) {
      float sine, cosine;
      sin_cos((double) pos, turns[i], sine, cosine);
      if (lane + 64 * i < half) angle[wave][lane + 64 * i] = make_float2(cosine * a.scale, sine * a.scale);
    }
  wave_order();
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const uint32_t e = g * 8 + j;
    c[j] = 1.0f, s[j] = 0.0f;
    if ((uint32_t) j < mine) {
      const float2 v = angle[wave][pairs ? e / 2 : e < half ? e : e - half];
      c[j] = v.x, s[j] = (pairs ? !(j & 1) : e < half) ? -v.y : v.y;
    }
  }
  uint8_t* to = nullptr;  // where the row's keys go
  if constexpr (DST != 0)
    if (id < pg.pages) to = pg.data + ((uint64_t) id * a.kv_heads * pg.page + ((uint32_t) pos & (pg.page - 1))) * a.dim * kv::size_of(DST);
  float* row = lds[wave];
  for (;;) {
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
      const uint32_t h = h0 + i * each * a.parts;
      float(&y)[8] = x[i];
      if (a.q_weight || a.k_weight) {
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j++) ss = __builtin_fmaf(y[j], y[j], ss);
        for (uint32_t o = 1; o < a.group; o <<= 1) ss += xor_lane(ss, (int) o);
        const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float) a.dim), a.eps)));
        const bool normed = h < a.heads ? a.q_weight != nullptr : h < turned && a.k_weight;
#pragma unroll
        for (int j = 0; j < 8; j++) y[j] = normed ? __fmul_rn(__fmul_rn(y[j], r), h < a.heads ? wq[j] : wk[j]) : y[j];
      }
      float z[8];
      if (pairs) {
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] = y[j ^ 1];
      } else {
        wave_order();
        *(kv::f32x4*) (row + lane * 8) = kv::f32x4{y[0], y[1], y[2], y[3]};
        *(kv::f32x4*) (row + lane * 8 + 4) = kv::f32x4{y[4], y[5], y[6], y[7]};
        wave_order();
        const float* head = row + (lane - g) * 8;
        if (half % 8 == 0) {
          const uint32_t e = g * 8 < half ? g * 8 + half : g * 8 < a.rot ? g * 8 - half : g * 8;
          const kv::f32x4 u = *(const kv::f32x4*) (head + e), v = *(const kv::f32x4*) (head + e + 4);
#pragma unroll
          for (int j = 0; j < 4; j++) z[j] = u[j], z[4 + j] = v[j];
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const uint32_t e = g * 8 + j;
            z[j] = head[e < half ? e + half : e < a.rot ? e - half : e];
          }
        }
      }
      const uint32_t n = h < turned ? mine : 0;
#pragma unroll
      for (int j = 0; j < 8; j++) y[j] = (uint32_t) j < n ? __builtin_fmaf(z[j], s[j], __fmul_rn(y[j], c[j])) : y[j];
      if (h < all && active) {
        if (h < a.heads) {
          store8_as(a.out_type, a.q_out + (t * a.q_out_stride + h * a.q_out_head + g * 8) * kv::size_of(a.out_type), y);
        } else if constexpr (DST == 0) {
          store8_as(a.out_type, a.k_out + (t * a.k_out_stride + (h - a.heads) * a.k_out_head + g * 8) * kv::size_of(a.out_type), y);
        } else if (to) {
          const bool second = h >= turned;
          const uint32_t hh = h - (second ? turned : a.heads);
          if (DST == OSMOS_F8 && pg.scale) kv::divide8(y, scale[i]);
          kv::store8<DST>(to + (second ? pg.plane : 0) + ((uint64_t) hh * pg.page * a.dim + g * 8) * kv::size_of(DST), y);
        }
      }
    }
    h0 += kAhead * each * a.parts;
    if (h0 - first >= all) break;  // (the whole wave: first is the lane's offset in the round)
    load(h0);
  }
}

template <uint32_t IN, int AHEAD>
auto rope_of(uint32_t dst) {
  return dst == 0 ? rope_kernel<IN, 0u, AHEAD> : dst == OSMOS_F16 ? rope_kernel<IN, OSMOS_F16, AHEAD>
         : dst == OSMOS_BF16 ? rope_kernel<IN, OSMOS_BF16, AHEAD> : rope_kernel<IN, OSMOS_F8, AHEAD>;
}

bool rope_launch(const OsmosRope* o, const int32_t* pos, const kv::Step& st, const Pages& pg, uint32_t dst, const void* v, uint64_t v_stride,
                 uint64_t v_head, hipStream_t s) {
  RopeArgs a = {o->turns, o->q_weight, o->k_weight, (const uint8_t*) o->q, (const uint8_t*) o->k, (const uint8_t*) v, (uint8_t*) o->q_out,
                (uint8_t*) o->k_out, o->q_stride, o->q_head, o->k_stride, o->k_head, v_stride, v_head, o->q_out_stride, o->q_out_head,
                o->k_out_stride, o->k_out_head, o->out_type, o->heads, o->kv_heads, o->n, o->dim, o->rot, o->layout, o->scale, o->eps,
                o->offset, 1, 1};
  while (a.group * 8 < a.dim) a.group *= 2;
  const uint32_t all = a.heads + a.kv_heads * (dst ? 2 : 1), rounds = (all * a.group + 63) / 64;
  // waves: a head a lane where the rows are few (one trip to memory); 4096 in all where they are more, since each makes the row's angles
  // again: 1024 / 2048 / 4096 / 8192 take 11.1 / 10.1 / 10.1 / 12.3 us for 700 rows of 48 heads of 128 floats, 12.2 / 12.2 / 10.9 /
  // 12.6 for 3510 bf16 rows of 40
  a.parts = 4096 / a.n < 1 ? 1 : 4096 / a.n < rounds ? 4096 / a.n : rounds;
  const uint64_t waves = (uint64_t) a.n * a.parts;
  if (!launches((waves + kRopeWaves - 1) / kRopeWaves, 64 * kRopeWaves)) return false;
  const uint32_t grid = (uint32_t) ((waves + kRopeWaves - 1) / kRopeWaves);
  const bool one = a.parts == rounds;
  auto* kernel = o->type == OSMOS_F32 ? one ? rope_of<OSMOS_F32, 1>(dst) : rope_of<OSMOS_F32, 4>(dst)
                 : o->type == OSMOS_F16 ? one ? rope_of<OSMOS_F16, 1>(dst) : rope_of<OSMOS_F16, 4>(dst)
                                        : one ? rope_of<OSMOS_BF16, 1>(dst) : rope_of<OSMOS_BF16, 4>(dst);
  kernel<<<grid, 64 * kRopeWaves, 0, s>>>(a, pos, st, pg);
  return hipGetLastError() == hipSuccess;
}

}  // namespace rows
}  // namespace osm

using namespace osm;

extern "C" OSM_API bool osmos_rope_turns(const OsmosRopeScaling* s, uint32_t rot, double* turns, float* scale) {
  return rows::turns_of(s, rot, turns, scale);
}

extern "C" OSM_API bool osmos_rope(const OsmosRope* a, const int32_t* pos, void* stream) {
  if (!rows::rope_ok(a, false) || !pos || !rows::aligned(pos, 4)) return false;
  return rows::rope_launch(a, pos, kv::Step{}, rows::Pages{}, 0, nullptr, 0, 0, (hipStream_t) stream);
}

extern "C" OSM_API bool osmos_rope_append(const OsmosRope* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step,
                                          const void* v, uint64_t v_stride, uint64_t v_head, void* stream) {
  if (!rows::rope_append_ok(a, kv, layer, step, v, v_stride, v_head)) return false;
  const uint64_t plane = kv::plane_bytes(kv);
  const rows::Pages pg = {(uint8_t*) kv->data + 2ull * layer * plane, kv->scale ? kv->scale + 2ull * layer * kv->heads : nullptr, kv->pages,
                          kv->page, plane};
  return rows::rope_launch(a, nullptr, kv::step_of(step), pg, kv->type, v, v_stride, v_head, (hipStream_t) stream);
}
