// libosmos MI355X - what the entry points of include/osmos_rows.h decide before they queue anything: what they refuse, and the
// rotary turns of a longer context. plain C++, so that the host can check it by itself.
#pragma once
#include <math.h>
#include <stdint.h>

#include "../../include/osmos_rows.h"
#include "attnhost.h"

namespace osm {
namespace rows {

inline bool aligned(const void* p, uint64_t by) { return (uintptr_t) p % by == 0; }
// values of `type` at p, whose rows are `stride` apart
inline bool rows_ok(const void* p, uint32_t type, uint64_t stride, uint32_t n, uint64_t row) {
  return p && aligned(p, kv::size_of(type)) && stride <= (1ull << 40) && (n == 1 || stride >= row);
}

// a launch has fewer than 2^32 threads
inline bool launches(uint64_t blocks, uint32_t threads) { return blocks && blocks * threads <= 0xFFFFFFFFull; }

inline bool norm_ok(const OsmosNorm* a) {
  if (!a || !a->n || a->n > 0x7FFFFFF0u || !a->dim || a->dim > OSMOS_NORM_MAX_DIM || !kv::row_type(a->type)) return false;
  if (!rows_ok(a->x, a->type, a->x_stride, a->n, a->dim)) return false;
  if (a->add && !rows_ok(a->add, a->type, a->add_stride, a->n, a->dim)) return false;
  if (a->sum && !rows_ok(a->sum, a->type, a->sum_stride, a->n, a->dim)) return false;
  if (a->n > 1 && a->sum && ((a->sum == a->x && a->sum_stride != a->x_stride) || (a->sum == a->add && a->sum_stride != a->add_stride))) return false;
  if (a->out && (!kv::row_type(a->out_type) || !rows_ok(a->out, a->out_type, a->out_stride, a->n, a->dim))) return false;
  if (a->weight && (!kv::row_type(a->weight_type) || !aligned(a->weight, kv::size_of(a->weight_type)))) return false;
  if (a->x16 && (a->dim % 16 || !aligned(a->x16, 16) || !a->overflow || !aligned(a->overflow, 4))) return false;
  if (!a->codes != !a->scales) return false;
  if (a->codes && (a->dim % 32 || !aligned(a->codes, 16) || !aligned(a->scales, 4))) return false;
  return (a->sum || a->out || a->x16 || a->codes) && a->eps >= 0.0f && a->eps <= 3.4e38f && a->offset - a->offset == 0.0f;
}

inline bool rope_ok(const OsmosRope* a, bool paged) {
  if (!a || !a->turns || !aligned(a->turns, 8) || !a->n || a->n > 0x7FFFFFF0u) return false;
  if (!a->dim || a->dim % 8 || a->dim > OSMOS_ATTN_MAX_DIM || !a->rot || a->rot % 2 || a->rot > a->dim) return false;
  if (a->layout != OSMOS_ROPE_HALVES && a->layout != OSMOS_ROPE_PAIRS) return false;
  if (!kv::row_type(a->type) || !kv::row_type(a->out_type) || !a->heads || a->heads > 4096 || a->kv_heads > 4096) return false;
  if (!(a->scale - a->scale == 0.0f) || !(a->eps >= 0.0f) || a->eps > 3.4e38f || !(a->offset - a->offset == 0.0f)) return false;
  if ((a->q_weight && !aligned(a->q_weight, 4)) || (a->k_weight && !aligned(a->k_weight, 4))) return false;
  struct Part {
    const void* p;
    uint64_t stride, head;
    uint32_t type, heads;
  };
  const Part parts[4] = {{a->q, a->q_stride, a->q_head, a->type, a->heads}, {a->q_out, a->q_out_stride, a->q_out_head, a->out_type, a->heads},
                         {a->k, a->k_stride, a->k_head, a->type, a->kv_heads}, {a->k_out, a->k_out_stride, a->k_out_head, a->out_type, a->kv_heads}};
  for (int i = 0; i < (!a->kv_heads ? 2 : paged ? 3 : 4); i++) {
    const Part& p = parts[i];
    if (!p.p || !aligned(p.p, 16) || p.stride > (1ull << 40) || p.head > (1ull << 40)) return false;
    if ((a->n > 1 && p.stride * kv::size_of(p.type) % 16) || (p.heads > 1 && p.head * kv::size_of(p.type) % 16)) return false;
    if (p.heads > 1 && p.head < a->dim) return false;
    if (a->n > 1 && p.stride < a->dim) return false;
  }
  // (in place: each head is read and written by the same lanes, so the rows have to be the same ones)
  if (a->q_out == a->q && (a->type != a->out_type || (a->n > 1 && a->q_stride != a->q_out_stride) || (a->heads > 1 && a->q_head != a->q_out_head)))
    return false;
  if (a->kv_heads && !paged && a->k_out == a->k &&
      (a->type != a->out_type || (a->n > 1 && a->k_stride != a->k_out_stride) || (a->kv_heads > 1 && a->k_head != a->k_out_head)))
    return false;
  return true;
}
inline bool rope_append_ok(const OsmosRope* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step, const void* v,
                           uint64_t v_stride, uint64_t v_head) {
  if (!rope_ok(a, true) || !kv::cache_ok(kv) || layer >= kv->layers || !kv::step_ok(step, true)) return false;
  if (a->kv_heads != kv->heads || a->dim != kv->dim || a->n != step->n_tok || !v || !aligned(v, 16)) return false;
  const uint64_t size = kv::size_of(a->type);
  if (v_stride > (1ull << 40) || v_head > (1ull << 40) || (a->n > 1 && (v_stride * size % 16 || v_stride < a->dim))) return false;
  return a->kv_heads == 1 || (v_head * size % 16 == 0 && v_head >= a->dim);
}

inline bool turns_of(const OsmosRopeScaling* s, uint32_t rot, double* turns, float* scale) {
  if (!s || !turns || !scale || !rot || rot % 2 || rot > OSMOS_ATTN_MAX_DIM || s->kind > OSMOS_ROPE_BANDS) return false;
  const double two_pi = 6.283185307179586476925286766559;
  if (!(s->base > 1.0) || !(s->base <= 1e30)) return false;
  if (s->kind != OSMOS_ROPE_PLAIN && (!(s->factor >= 1.0) || !(s->factor <= 1e6))) return false;
  const bool ramp = s->kind == OSMOS_ROPE_YARN || s->kind == OSMOS_ROPE_BANDS;
  if (ramp && (!(s->context >= 1.0) || !(s->context <= 1e12) || !(s->low > 0.0) || !(s->high > s->low) || !(s->high <= 1e12))) return false;
  if (s->kind == OSMOS_ROPE_NTK && rot < 4) return false;
  const double base = s->kind == OSMOS_ROPE_NTK ? s->base * pow(s->factor, rot / (rot - 2.0)) : s->base;
  *scale = s->kind == OSMOS_ROPE_YARN ? (float) (0.1 * log(s->factor) + 1.0) : 1.0f;
  // YARN: the pair that makes so many turns in the context, as a (broken) number of pairs
  double first = 0, last = 0;
  if (s->kind == OSMOS_ROPE_YARN) {
    const double at = rot / (2.0 * log(base));
    first = floor(at * log(s->context / (two_pi * s->high))), last = ceil(at * log(s->context / (two_pi * s->low)));
    first = first < 0 ? 0 : first, last = last > rot - 1.0 ? rot - 1.0 : last;
    if (last <= 0) first = -1, last = 0;  // (a context so short that the first pair makes no more than `slow`: all divided)
    if (last - first < 0.001) last = first + 0.001;
  }
  for (uint32_t i = 0; i < rot / 2; i++) {
    double f = pow(base, -2.0 * i / rot);
    if (s->kind == OSMOS_ROPE_LINEAR) f /= s->factor;
    if (ramp) {
      double slow = s->kind == OSMOS_ROPE_YARN ? (i - first) / (last - first)
                                               : 1.0 - (s->context * f / two_pi - s->low) / (s->high - s->low);
      slow = slow < 0 ? 0 : slow > 1 ? 1 : slow;
      f = f * (1.0 - slow) + f / s->factor * slow;
    }
    turns[i] = f / two_pi;
  }
  return true;
}

inline bool sample_ok(const OsmosSample* a) {
  if (!a || !a->n || a->n > 0x7FFFFFu || !a->vocab || a->vocab > OSMOS_SAMPLE_MAX_VOCAB || !kv::row_type(a->type) ||
      (uint64_t) a->n * a->vocab > 1ull << 40)
    return false;
  if (!rows_ok(a->logits, a->type, a->stride, a->n, a->vocab) || !a->u || !a->token) return false;
  const void* words[] = {a->u, a->temperature, a->top_p, a->min_p, a->top_k, a->token, a->prob, a->kept, a->probs};
  for (const void* p : words)
    if (!aligned(p, 4)) return false;
  return true;
}

}  // namespace rows
}  // namespace osm
