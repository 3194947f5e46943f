// libosmos MI355X - what the paged cache's kernels and the attention share (include/osmos_attn.h): 8 values at a time in
// the cache's and the callers' types, and a step's sequences as the device memory says they are, clamped so that no table
// leads a kernel out of its buffers.
#pragma once
#include "attnhost.h"
#include "common.h"

namespace osm {
namespace kv {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 8 consecutive values as floats
template <uint32_t T>
__device__ inline void load8(const void* p, float (&x)[8]) {
  if constexpr (T == OSMOS_F32) {
    const f32x4 a = gload<f32x4>(p), b = gload<f32x4>((const f32x4*) p + 1);
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
  } else if constexpr (T == OSMOS_F16) {
    const f16x8 a = gload<f16x8>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float) a[i];
  } else {
    const bf16x8 a = gload<bf16x8>(p);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float) a[i];
  }
}

// e4m3 of two floats, nearest with ties to even: the conversion makes NaN of what is past 448, so that is clamped first;
// a NaN passes the clamp (med3 of a NaN is not one)
__device__ inline float f8_clamp(float x) { return x != x ? x : __builtin_amdgcn_fmed3f(x, -448.0f, 448.0f); }
__device__ inline uint32_t f8_word(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(f8_clamp(a), f8_clamp(b), 0, false);
  return (uint32_t) __builtin_amdgcn_cvt_pk_fp8_f32(f8_clamp(c), f8_clamp(d), w, true);
}

template <uint32_t T>
__device__ inline void store8(void* p, const float (&x)[8]) {
  if constexpr (T == OSMOS_F32) {
    *(f32x4*) p = f32x4{x[0], x[1], x[2], x[3]};
    *((f32x4*) p + 1) = f32x4{x[4], x[5], x[6], x[7]};
  } else if constexpr (T == OSMOS_F16) {
    f16x8 r;
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = (_Float16) x[i];
    *(f16x8*) p = r;
  } else if constexpr (T == OSMOS_BF16) {
    bf16x8 r;
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = (__bf16) x[i];
    *(bf16x8*) p = r;
  } else {
    *(u32x2*) p = u32x2{f8_word(x[0], x[1], x[2], x[3]), f8_word(x[4], x[5], x[6], x[7])};
  }
}

// a step's tables with their bounds
struct Step {
  const int32_t *start, *len, *table, *seq, *live;
  uint32_t n_seq, n_tok, max_len, seqs, width;  // width: table_stride
};

struct Seq {
  int row0, rows;        // its rows in the step
  int len;               // its tokens, the rows' among them (none where it takes no part in the step)
  int end;               // the tokens that may be read: len within the table's room and max_len
  const int32_t* table;  // its pages (paged only)
};

__device__ inline int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// sequence s as the step's tables give it. page 0: packed rows (its tokens are its rows)
__device__ inline Seq sequence(const Step& st, uint32_t s, uint32_t page) {
  Seq q;
  q.row0 = clampi(st.start[s], 0, (int) st.n_tok);
  q.rows = clampi(st.start[s + 1], q.row0, (int) st.n_tok) - q.row0;
  q.len = q.end = q.rows;
  q.table = nullptr;
  if (page) {
    const uint32_t id = st.seq ? (uint32_t) st.seq[s] : s;
    if (id >= st.seqs) {
      q.rows = q.len = q.end = 0;
      return q;
    }
    const uint64_t room = (uint64_t) st.width * page;
    const bool live = !st.live || st.live[s];
    q.len = live ? clampi(st.len[id], 0, 0x7FFFFFFF) : 0;
    q.end = clampi(q.len, 0, room < st.max_len ? (int) room : (int) st.max_len);
    q.table = st.table + (uint64_t) id * st.width;
  }
  return q;
}

// lane `at`'s sequence, for the whole wave
__device__ inline int lane_of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ inline Seq lane_of(const Seq& q, int at) {
  Seq r;
  r.row0 = lane_of(q.row0, at), r.rows = lane_of(q.rows, at), r.len = lane_of(q.len, at), r.end = lane_of(q.end, at);
  r.table = (const int32_t*) ((uint64_t) (uint32_t) lane_of((int) ((uint64_t) q.table >> 32), at) << 32 |
                              (uint32_t) lane_of((int) (uint64_t) q.table, at));
  return r;
}

// the sequence of row t, the last one that starts at or before it; false for none. the whole wave asks for one t: up to 64
// sequences are read whole at once, a lane each, so that no load waits for the search; more by their starts, 64 a round. all 64
// lanes have to be active: one that is not hides its sequence
__device__ inline bool sequence_of(const Step& st, int t, uint32_t page, Seq& q) {
  const uint32_t lane = threadIdx.x & 63;
  if (st.n_seq <= 64) {
    const Seq mine = sequence(st, lane < st.n_seq ? lane : 0, page);
    const uint64_t at = __ballot(lane < st.n_seq && st.start[lane < st.n_seq ? lane : 0] <= t);
    if (!at) return false;
    q = lane_of(mine, 63 - __builtin_clzll(at));
    return true;
  }
  uint32_t lo = 0, n = st.n_seq;
  for (;;) {
    const uint32_t by = (n + 63) / 64, i = lane * by;
    const uint64_t at = __ballot(i < n && st.start[lo + (i < n ? i : 0)] <= t);
    const int c = __popcll(at);
    if (c == 0) return false;
    lo += (uint32_t) (c - 1) * by;
    n = by < n - (uint32_t) (c - 1) * by ? by : n - (uint32_t) (c - 1) * by;
    if (by == 1) break;
  }
  q = sequence(st, lo, page);
  return true;
}

inline Step step_of(const OsmosKvStep* st) {
  return Step{st->start, st->len, st->table, st->seq, st->live, st->n_seq, st->n_tok, st->max_len, st->seqs, st->table_stride};
}

}  // namespace kv
}  // namespace osm
