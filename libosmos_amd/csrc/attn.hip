// libosmos MI355X - attention over packed rows and over the paged cache (include/osmos_attn.h).
//
// a row's output is sum_j p_j v_j / sum_j p_j with p_j = exp(scale q k_j - m), m the greatest score, in one pass: the
// running m and sum, the sum and output scaled by exp(m_old - m_new) where m grows.
#include "kvcache.h"

namespace osm {
namespace attn {

using kv::Seq;
using kv::Step;
using kv::sequence;
using kv::sequence_of;

struct Args {
  const uint8_t* q;
  uint8_t* out;
  float* lse;
  uint64_t qs, qh, os, oh;
  uint32_t q_type, out_type, heads, group, window, dim;
  float scale;
};

// keys and values: packed rows (page 0), or a layer's two planes of pages
struct Kv {
  const uint8_t *k, *v;
  uint64_t ks, kh, vs, vh;  // packed: strides of a row and a head
  uint32_t type, page, pages, heads;
  const float* scale;
};

__device__ inline float value(uint32_t type, const uint8_t* p, uint64_t i) {
  if (type == OSMOS_F32) return ((const float*) p)[i];
  if (type == OSMOS_F16) return (float) ((const _Float16*) p)[i];
  if (type == OSMOS_BF16) return (float) ((const __bf16*) p)[i];
  return __builtin_amdgcn_cvt_f32_fp8(p[i], 0);
}

// a wave a row and head: 64 keys a round, a key a lane for the scores, a dim a lane (in turns of 64) for the output
__global__ __launch_bounds__(64) void row_kernel(Args a, Kv kv, Step st) {
  __shared__ float qv[OSMOS_ATTN_MAX_DIM];
  const uint32_t t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, g = h / a.group;
  const int s = sequence_of(st, (int) t);
  if (s < 0) return;
  const Seq seq = sequence(st, (uint32_t) s, kv.page);
  if ((int) t < seq.row0 || (int) t >= seq.row0 + seq.rows) return;
  const int pos = seq.len - (seq.row0 + seq.rows - (int) t);
  const int end = pos + 1 < seq.end ? pos + 1 : seq.end;
  const int begin = a.window && pos + 1 > (int) a.window ? pos + 1 - (int) a.window : 0;
  const bool bf = kv.type == OSMOS_BF16 || (kv.type == OSMOS_F8 && a.q_type == OSMOS_BF16);  // the products' type
  for (uint32_t d = lane; d < a.dim; d += 64) {
    const float x = value(a.q_type, a.q, t * a.qs + h * a.qh + d);
    qv[d] = bf ? (float) (__bf16) x : (float) (_Float16) x;
  }
  __syncthreads();
  const float ks = kv.scale ? kv.scale[g] : 1.0f, vs = kv.scale ? kv.scale[kv.heads + g] : 1.0f;
  float m = -__builtin_inff(), l = 0.0f, o[4] = {};
  for (int j0 = begin; j0 < end; j0 += 64) {
    const int j = j0 + (int) lane;
    bool in = j < end;
    uint64_t kat = 0, vat = 0;
    if (in) {
      if (kv.page) {
        const uint32_t id = (uint32_t) seq.table[(uint32_t) j / kv.page];
        in = id < kv.pages;
        kat = vat = (((uint64_t) id * kv.heads + g) * kv.page + (uint32_t) j % kv.page) * a.dim;
      } else {
        kat = (uint64_t) (seq.row0 + j) * kv.ks + g * kv.kh, vat = (uint64_t) (seq.row0 + j) * kv.vs + g * kv.vh;
      }
    }
    float x = 0.0f;
    if (in)
      for (uint32_t d = 0; d < a.dim; d++) x = __builtin_fmaf(qv[d], value(kv.type, kv.k, kat + d), x);
    x = in ? x * (a.scale * ks) : -__builtin_inff();
    float top = x;
    for (int o2 = 1; o2 < 64; o2 <<= 1) top = fmaxf(top, __shfl_xor(top, o2));
    top = fmaxf(top, m);
    if (top == -__builtin_inff()) continue;
    const float p = in ? expf(x - top) : 0.0f, c = expf(m - top);
    float sum = p;
    for (int o2 = 1; o2 < 64; o2 <<= 1) sum += __shfl_xor(sum, o2);
    l = l * c + sum, m = top;
    for (int i = 0; i < 4; i++) o[i] *= c;
    for (int i = 0; i < 64; i++) {
      if (!__shfl((int) in, i)) continue;
      const float pi = __shfl(p, i);
      const uint64_t at = ((uint64_t) (uint32_t) __shfl((int) (vat >> 32), i) << 32) | (uint32_t) __shfl((int) vat, i);
      for (int e = 0; e < 4; e++)
        if (lane + 64 * e < a.dim) o[e] = __builtin_fmaf(pi, value(kv.type, kv.v, at + lane + 64 * e), o[e]);
    }
  }
  for (int e = 0; e < 4; e++) {
    const uint32_t d = lane + 64 * e;
    if (d >= a.dim) break;
    const float y = l > 0.0f ? o[e] * vs / l : l == 0.0f ? 0.0f : l;
    const uint64_t at = t * a.os + h * a.oh + d;
    if (a.out_type == OSMOS_F32) ((float*) a.out)[at] = y;
    else if (a.out_type == OSMOS_F16) ((_Float16*) a.out)[at] = (_Float16) y;
    else ((__bf16*) a.out)[at] = (__bf16) y;
  }
  if (a.lse && lane == 0) a.lse[(uint64_t) t * a.heads + h] = m + logf(l);
}

inline bool row_type(uint32_t t) { return t == OSMOS_F32 || t == OSMOS_F16 || t == OSMOS_BF16; }
inline bool stride_ok(uint64_t stride, uint32_t type) { return stride * kv::size_of(type) % 16 == 0; }

inline bool args_ok(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim) {
  if (!a || !a->q || !a->out || (uintptr_t) a->q % 16 || (uintptr_t) a->out % 16) return false;
  if (!row_type(a->q_type) || !row_type(a->out_type) || !a->heads || a->heads > 4096 || a->heads % kv_heads) return false;
  if (!stride_ok(a->q_stride, a->q_type) || !stride_ok(a->q_head, a->q_type) || !stride_ok(a->out_stride, a->out_type) ||
      !stride_ok(a->out_head, a->out_type))
    return false;
  return a->window <= 0x7FFFFFFFu && a->scale == a->scale && dim;
}
inline Args args_of(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim) {
  return Args{(const uint8_t*) a->q, (uint8_t*) a->out, a->lse, a->q_stride, a->q_head, a->out_stride, a->out_head,
              a->q_type, a->out_type, a->heads, a->heads / kv_heads, a->window, dim, a->scale};
}
inline Kv pages_of(const OsmosKv* kv, uint32_t layer) {
  const uint64_t plane = (uint64_t) kv->pages * kv->heads * kv->page * kv->dim * kv::size_of(kv->type);
  const uint8_t* k = (const uint8_t*) kv->data + 2ull * layer * plane;
  return Kv{k, k + plane, 0, 0, 0, 0, kv->type, kv->page, kv->pages, kv->heads,
            kv->scale ? kv->scale + 2ull * layer * kv->heads : nullptr};
}

bool run_rows(const OsmosAttn* a, const Kv& k, uint32_t dim, const OsmosKvStep* step, void* stream) {
  row_kernel<<<dim3(step->n_tok, a->heads), 64, 0, (hipStream_t) stream>>>(args_of(a, k.heads, dim), k, kv::step_of(step));
  return hipGetLastError() == hipSuccess;
}

}  // namespace attn
}  // namespace osm

using namespace osm;

extern "C" OSM_API uint64_t osmos_attn_workspace(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim,
                                                 const OsmosKvStep* step) {
  (void) a, (void) kv_heads, (void) dim, (void) step;
  return 0;
}

extern "C" OSM_API bool osmos_attn_prompt(const OsmosAttn* a, const OsmosKvRows* r, const OsmosKvStep* step,
                                          void* workspace, uint64_t workspace_bytes, void* stream) {
  (void) workspace, (void) workspace_bytes;
  if (!r || !r->k || !r->v || !r->heads || r->heads > 4096 || (r->type != OSMOS_F16 && r->type != OSMOS_BF16)) return false;
  if (!r->dim || r->dim > OSMOS_ATTN_MAX_DIM || r->dim % 16 || (uintptr_t) r->k % 16 || (uintptr_t) r->v % 16) return false;
  if (r->k_stride % 8 || r->k_head % 8 || r->v_stride % 8 || r->v_head % 8) return false;
  if (!attn::args_ok(a, r->heads, r->dim) || !kv::step_ok(step, false)) return false;
  const attn::Kv k{(const uint8_t*) r->k, (const uint8_t*) r->v, r->k_stride, r->k_head, r->v_stride, r->v_head, r->type,
                   0, 0, r->heads, nullptr};
  return attn::run_rows(a, k, r->dim, step, stream);
}

extern "C" OSM_API bool osmos_attn_chunk(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step,
                                         void* workspace, uint64_t workspace_bytes, void* stream) {
  (void) workspace, (void) workspace_bytes;
  if (!kv::cache_ok(kv) || layer >= kv->layers || !attn::args_ok(a, kv->heads, kv->dim) || !kv::step_ok(step, true)) return false;
  return attn::run_rows(a, attn::pages_of(kv, layer), kv->dim, step, stream);
}

extern "C" OSM_API bool osmos_attn_token(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step,
                                         void* workspace, uint64_t workspace_bytes, void* stream) {
  (void) workspace, (void) workspace_bytes;
  if (!kv::cache_ok(kv) || layer >= kv->layers || !attn::args_ok(a, kv->heads, kv->dim) || !kv::step_ok(step, true)) return false;
  if (step->max_tok != 1) return false;
  return attn::run_rows(a, attn::pages_of(kv, layer), kv->dim, step, stream);
}
