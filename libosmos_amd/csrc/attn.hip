// libosmos MI355X - attention over packed rows and over the paged cache (include/osmos_attn.h).
//
// a row's output is sum_j p_j v_j / sum_j p_j with p_j = exp(scale q k_j - m), m the greatest score, in one pass: the
// running m and sum, the sum and output scaled by exp(m_old - m_new) where m grows. scores, sums, maxima and outputs are
// kept in float; the p_j are rounded to the products' 16-bit type, as the matrix units take no other: an error of the size of a
// 16-bit output's own rounding and independent of it (a bf16 prompt of 8192 is 2.2e-3 off in all, relative, where the
// output's rounding alone makes 1.6e-3). the sum takes the p_j before that. f16 has no values between 0 and 2^-24, and
// thousands of keys of less weight than that count together: its p_j are taken 2^lift times as large, up to 2^15, by a running m
// that is the greatest score less the lift (in powers of two), and the factor leaves sum and output at the end. a tile's p_j are
// summed before they join the running sum, which one by one would not notice those below 2^-24 of it.
#include <type_traits>

#include "kvcache.h"

namespace osm {
namespace attn {

using kv::Seq;
using kv::Step;
using kv::lane_of;
using kv::sequence;

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

// ---- the two 16-bit types the products are taken in ----
typedef kv::f32x4 f32x4;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef kv::u32x2 u32x2;
typedef kv::u32x4 u32x4;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <bool BF> struct Unit;
template <> struct Unit<false> {
  typedef _Float16 e;
  typedef kv::f16x8 v8;
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  static constexpr int kLift = 15;  // p_j up to 2 to this
  static __device__ inline f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ inline f32x16 mfma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ inline f16x2 f8_low(uint32_t w) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int) w, 1.0f, false); }
  static __device__ inline f16x2 f8_high(uint32_t w) { return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int) w, 1.0f, true); }
};
template <> struct Unit<true> {
  typedef __bf16 e;
  typedef kv::bf16x8 v8;
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  static constexpr int kLift = 0;
  static __device__ inline f32x4 mfma16(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ inline f32x16 mfma32(v8 a, v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ inline bf16x2 f8_low(uint32_t w) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int) w, 1.0f, false); }
  static __device__ inline bf16x2 f8_high(uint32_t w) { return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int) w, 1.0f, true); }
};

// 8 e4m3 values (two words) in the products' type: exact in either
template <bool BF>
__device__ inline typename Unit<BF>::v8 from_f8(u32x2 w) {
  typename Unit<BF>::v8 r;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const auto a = Unit<BF>::f8_low(w[i]), b = Unit<BF>::f8_high(w[i]);
    r[4 * i] = a[0], r[4 * i + 1] = a[1], r[4 * i + 2] = b[0], r[4 * i + 3] = b[1];
  }
  return r;
}

// a lane's values of a query head as the B operand of N steps, 8 dims each from at(i) on, in the products' type (an F32 q's
// rounded once), negated for a negative scale; zeros where `in` is false, past the
// dims and for a scale of 0
template <bool BF, int N, uint32_t T, class At>
__device__ inline void q_steps(const uint8_t* p, uint32_t dim, bool in, float sign, At at, typename Unit<BF>::v8 (&q)[N]) {
  float x[N][8];
#pragma unroll
  for (int i = 0; i < N; i++) kv::load8<T>(p + (at(i) < dim ? at(i) : 0) * kv::size_of(T), x[i]);
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float f = in && at(i) < dim ? sign : 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) q[i][j] = f == 0.0f ? (typename Unit<BF>::e) 0.0f : (typename Unit<BF>::e) (x[i][j] * f);
  }
}
template <bool BF, int N, class At>
__device__ inline void load_q(const Args& a, uint64_t row, uint32_t head, bool in, float scale, At at,
                              typename Unit<BF>::v8 (&q)[N]) {
  const uint8_t* p = a.q + (row * a.qs + head * a.qh) * kv::size_of(a.q_type);
  const float sign = scale < 0.0f ? -1.0f : scale == 0.0f ? 0.0f : 1.0f;
  if (a.q_type == OSMOS_F32) q_steps<BF, N, OSMOS_F32>(p, a.dim, in, sign, at, q);
  else if (a.q_type == OSMOS_F16) q_steps<BF, N, OSMOS_F16>(p, a.dim, in, sign, at, q);
  else q_steps<BF, N, OSMOS_BF16>(p, a.dim, in, sign, at, q);
}

__device__ inline void put4(const Args& a, uint64_t at, f32x4 y) {
  if (a.out_type == OSMOS_F32) {
    *(f32x4*) (a.out + at * 4) = y;
  } else if (a.out_type == OSMOS_F16) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *(h4*) (a.out + at * 2) = h4{(_Float16) y[0], (_Float16) y[1], (_Float16) y[2], (_Float16) y[3]};
  } else {
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    *(b4*) (a.out + at * 2) = b4{(__bf16) y[0], (__bf16) y[1], (__bf16) y[2], (__bf16) y[3]};
  }
}

// the greatest (or the sum) over the four lanes that share lane % 16
__device__ inline float max_rows(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}
__device__ inline float sum_rows(float x) {
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = __int_as_float(a[0]) + __int_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return __int_as_float(b[0]) + __int_as_float(b[1]);
}

constexpr float kLog2E = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
// what a score is multiplied with (its sign is in q; of a scale of 0 q is zeros, as -infinity times 0 would be NaN)
__device__ inline float unit_of(float scale) { return scale == 0.0f ? 1.0f : fabsf(scale) * kLog2E; }
// a maximum as what is subtracted: of nothing (-infinity), zero, so that exp2 of the difference is 0 and not NaN
__device__ inline float finite_max(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// ---- one row a sequence (osmos_attn_token) ----
// scores and outputs are computed transposed, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_16x16x32 with up to 16 of a kv
// head's query heads as columns: then a lane holds one query head's scores (of 8 keys of a tile of 32), its maximum, sum
// and scaling are the lane's own, and the accumulator's layout of P^T is the B operand's of the second product but for the
// order of the keys, which the V rows' order takes up. K goes straight from memory into the A operand's registers (a lane
// 16 bytes of one key's row); V passes through the wave's own LDS tile, as its columns are wanted: written as it lies
// (16-byte pieces turned by row so that the transposing reads meet no bank twice), read by ds_read_tr.
// a workgroup is 4 waves over one chunk of a sequence's keys for one kv head; wave w takes the tiles w, w + 4, ..: no
// barrier until the waves' results are joined. the next tile's rows are loaded while this one is worked on, and the page
// ids of the one after. with pages of 16 tokens or more (WIDE) half a tile lies in one page, so that its place is the
// wave's and not a lane's: scalar loads and arithmetic, where smaller pages take some 60 vector instructions a tile.
// no load is conditional: a place that is masked reads a row that exists and its score and value are then replaced.
// bound by memory: one sequence of 131072 tokens (8 kv heads of 128, bf16) 93 us for 537 MB, 5.8 TB/s (a
// streaming read reaches 7.2). a short step is a chain of loads: lengths, page ids, rows, some 1.7 us a tile of a wave's.
// two tiles in flight a wave instead of one (244 registers) measured the same, three workgroups a compute unit (10 spilled
// registers) 14 % slower.
template <bool F8, int D> struct TokenTile {
  static constexpr int kSize = F8 ? 1 : 2;
  static constexpr int kRow = D * kSize;                        // bytes of a V row in LDS
  static constexpr int kPieces = kRow / 64;                     // 16-byte pieces a lane loads of a row
  static constexpr int kOut = 16 * (D + 4) * 4;                 // a wave's result for the join
  static constexpr int kLds = 32 * kRow > kOut ? 32 * kRow : kOut;
  // the place of piece c of row r
  static __device__ inline int at(int r, int c) {
    constexpr int pieces = kRow / 16, rows = kRow < 256 ? 256 / kRow : 1;
    const int turn = F8 ? r / rows : 2 * (r / rows);
    return r * kRow + ((c ^ (turn & (pieces < 16 ? pieces - 1 : 15))) * 16);
  }
};

// the keys of a sequence's row from the first tile on that its window reaches
__device__ inline int first_key(const Seq& q, uint32_t window) { return window && q.len > (int) window ? q.len - (int) window : 0; }
__device__ inline int keys_of(const Seq& q, uint32_t window) {
  const int n = q.end - (first_key(q, window) & ~31);
  return q.rows < 1 || n < 0 ? 0 : n;
}

// the sum of x over this lane and those below it
__device__ inline uint32_t wave_scan(uint32_t x) {
#define OSM_ADD_DPP(ctrl, rows) x += (uint32_t) __builtin_amdgcn_update_dpp(0, (int) x, ctrl, rows, 0xF, false)
  OSM_ADD_DPP(0x111, 0xF);  // row_shr 1, 2, 4, 8
  OSM_ADD_DPP(0x112, 0xF);
  OSM_ADD_DPP(0x114, 0xF);
  OSM_ADD_DPP(0x118, 0xF);
  OSM_ADD_DPP(0x142, 0xA);  // row_bcast 15, 31
  OSM_ADD_DPP(0x143, 0xC);
#undef OSM_ADD_DPP
  return x;
}

// the step's work cut into chunks (chunk_keys): workgroup `index` takes chunk c of sequence s's n. every workgroup reads all
// lengths, 64 a round, and finds its place by their running sum, as no one else knows them; at most want + n_seq chunks.
struct Work {
  uint32_t s, c, n, chunk;
  Seq seq;
};
__device__ inline bool find_work(const Step& st, uint32_t page, uint32_t window, uint32_t want, uint32_t index, Work& w) {
  const uint32_t lane = threadIdx.x & 63;
  Seq none, q;
  none.row0 = none.rows = none.len = none.end = 0, none.table = st.table;
  uint32_t total = 0;  // in tiles of 32
  q = lane < st.n_seq ? sequence(st, lane, page) : none;
  for (uint32_t s = 0;;) {
    total += (uint32_t) lane_of((int) wave_scan(((uint32_t) keys_of(q, window) + 31) / 32), 63);
    if ((s += 64) >= st.n_seq) break;
    q = s + lane < st.n_seq ? sequence(st, s + lane, page) : none;
  }
  w.chunk = chunk_keys(total, want);
  uint32_t before = 0;
  for (uint32_t s = 0; s < st.n_seq; s += 64) {
    if (st.n_seq > 64) q = s + lane < st.n_seq ? sequence(st, s + lane, page) : none;
    const int k = keys_of(q, window);
    const uint32_t n = q.rows < 1 ? 0 : chunks_of(k, w.chunk), x = before + wave_scan(n);
    const uint64_t past = __ballot(x > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      w.s = s + (uint32_t) at;
      w.n = (uint32_t) lane_of((int) n, at);
      w.c = index - ((uint32_t) lane_of((int) x, at) - w.n);
      w.seq = lane_of(q, at);
      return true;
    }
    before = (uint32_t) lane_of((int) x, 63);
  }
  return false;
}

// a word of a table at a place that is the whole wave's
__device__ inline int uniform_word(const int32_t* p) {
  return *(const __attribute__((address_space(4))) int32_t*) (uint64_t) p;
}

template <bool BF, bool F8, int D, bool WIDE>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void token_kernel(Args a, Kv kv, Step st, uint32_t want, uint32_t tiles,
                                                                   uint32_t* __restrict__ cut, float* __restrict__ part) {
  typedef Unit<BF> U;
  typedef typename U::v8 v8;
  typedef TokenTile<F8, D> T;
  constexpr int kSteps = D / 32, kDims = D / 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds[4][T::kLds];
  __shared__ float ml[4][2][16];
  const uint32_t lane = threadIdx.x & 63, wave = (uint32_t) __builtin_amdgcn_readfirstlane((int) threadIdx.x / 64);
  const uint32_t r = lane & 15, quad = lane / 16;
  uint32_t b = blockIdx.x;
  const uint32_t mt = b % tiles;
  b /= tiles;
  const uint32_t g = b % kv.heads;
  b /= kv.heads;
  Work work;
  if (!find_work(st, kv.page, a.window, want, b, work)) return;
  const uint32_t s = work.s;
  const Seq seq = work.seq;
  const int begin = first_key(seq, a.window), from = (begin & ~31) + (int) (work.c * work.chunk);
  const int to = seq.end - from > (int) work.chunk ? from + (int) work.chunk : seq.end;
  if (cut && work.c == 0 && g == 0 && mt == 0 && threadIdx.x == 0) cut[2 * s] = b, cut[2 * s + 1] = work.n;
  const uint32_t row = (uint32_t) (seq.row0 + seq.rows - 1);
  const uint32_t heads = a.group - mt * 16 < 16 ? a.group - mt * 16 : 16, head0 = g * a.group + mt * 16;

  // the rows of a tile that a lane loads are 16 i + r, their 16-byte pieces 4 p + quad
  const uint32_t dim_bytes = a.dim * T::kSize, shift = 31 - __builtin_clz(kv.page);
  const uint64_t page_bytes = (uint64_t) kv.heads * kv.page * dim_bytes, head_at = (uint64_t) g * kv.page * dim_bytes;
  uint32_t piece[T::kPieces];
#pragma unroll
  for (int p = 0; p < T::kPieces; p++) {
    const uint32_t d = 64 * p + 16 * quad;
    piece[p] = (WIDE ? r * dim_bytes : 0) + (d < dim_bytes ? d : 0);
  }
  int id[2];
  auto ids = [&](int j0) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int j = j0 + 16 * i + (WIDE ? 0 : (int) r), last = to - 1;
      const int32_t* at = seq.table + ((uint32_t) (j < last ? j : last) >> shift);
      id[i] = WIDE ? uniform_word(at) : gload<int>(at);
    }
  };
  u32x4 kr[2][T::kPieces], vr[2][T::kPieces];
  bool page_in[2];
  auto load = [&](int j0) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      page_in[i] = (uint32_t) id[i] < kv.pages;
      const uint32_t slot = (uint32_t) (j0 + 16 * i + (WIDE ? 0 : (int) r)) & (kv.page - 1);
      const uint64_t at = (page_in[i] ? (uint32_t) id[i] : 0u) * page_bytes + head_at + slot * dim_bytes;
      const uint8_t *k = kv.k + at, *v = kv.v + at;
#pragma unroll
      for (int p = 0; p < T::kPieces; p++) kr[i][p] = gload<u32x4>(k + piece[p]);
#pragma unroll
      for (int p = 0; p < T::kPieces; p++) vr[i][p] = gload<u32x4>(v + piece[p]);
    }
  };

  const int first = from + 32 * (int) wave;
  if (first < to) ids(first);

  // Q^T as the B operand: column lane % 16, 8 dims a lane of each step's 32; of 8-bit keys a lane loads 16 dims at once,
  // so that two steps share 64 dims
  v8 q[kSteps];
  const float scale = a.scale * (F8 && kv.scale ? kv.scale[g] : 1.0f), unit = unit_of(scale);
  load_q<BF, kSteps>(a, row, head0 + (r < heads ? r : 0), r < heads, scale, [&](int i) {
    return F8 ? (uint32_t) (64 * (i / 2) + 16 * quad + 8 * (i % 2)) : (uint32_t) (32 * i + 8 * quad);
  }, q);

  f32x4 o[kDims];
#pragma unroll
  for (int i = 0; i < kDims; i++) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = -__builtin_inff(), l = 0.0f;

  uint8_t* tile = lds[wave];
  if (first < to) {
    load(first);
    ids(first + 128);
  }
  for (int j0 = first; j0 < to; j0 += 128) {
    // the tile's keys that are there, a bit each
    uint32_t live = 0xFFFFFFFFu;
    if (WIDE) {
      if (!page_in[0]) live &= 0xFFFF0000u;
      if (!page_in[1]) live &= 0x0000FFFFu;
    } else {
      live = ((uint32_t) __ballot(page_in[0]) & 0xFFFFu) | (uint32_t) __ballot(page_in[1]) << 16;
    }
    if (j0 + 32 > to) live &= (1u << (to - j0)) - 1;
    if (j0 < begin) live &= 0xFFFFFFFFu << (begin - j0);
    if (live != 0xFFFFFFFFu) {  // (zeros for the others' values: what lies there has no influence)
#pragma unroll
      for (int i = 0; i < 2; i++)
        if (!(live >> (16 * i + r) & 1)) {
#pragma unroll
          for (int p = 0; p < T::kPieces; p++) vr[i][p] = u32x4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int p = 0; p < T::kPieces; p++) *(u32x4*) (tile + T::at(16 * i + r, 4 * p + quad)) = vr[i][p];
    // S^T: two tiles of 16 keys
    f32x4 x[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      x[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (a.dim < D) {  // (the piece read in place of one past the dims)
#pragma unroll
        for (int p = 0; p < T::kPieces; p++)
          if (64 * p + 16 * quad >= dim_bytes) kr[i][p] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int k = 0; k < kSteps; k++) {
        v8 ka;
        if constexpr (F8) ka = from_f8<BF>(u32x2{kr[i][k / 2][2 * (k % 2)], kr[i][k / 2][2 * (k % 2) + 1]});
        else ka = __builtin_bit_cast(v8, kr[i][k]);
        x[i] = U::mfma16(ka, q[k], x[i]);
      }
    }
    if (j0 + 128 < to) {
      load(j0 + 128);
      ids(j0 + 256);
    }
    __builtin_amdgcn_sched_barrier(0);  // (the loads go out before the softmax)
    if (live != 0xFFFFFFFFu) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
          if (!(live >> (16 * i + 4 * quad + j) & 1)) x[i][j] = -__builtin_inff();
    }
    float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])), fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
    top = fmaxf(m, __builtin_fmaf(max_rows(top), unit, -(float) U::kLift));
    const float base = finite_max(top);
    if (__any(top > m)) {  // (seldom, once the greatest scores have been met)
      const float fade = __builtin_amdgcn_exp2f(m - base);
      m = top;
      l *= fade;
#pragma unroll
      for (int t = 0; t < kDims; t++) o[t] *= fade;
    }
    v8 p;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][j], unit, -base));
        sum = i + j ? sum + e : e;
        p[4 * i + j] = (typename U::e) e;
      }
    l += sum;
    // O^T: V^T's columns of keys 4 quad + 0 .. 3 and 16 + 4 quad + 0 .. 3, as P^T's lanes hold them
#pragma unroll
    for (int t = 0; t < kDims; t++) {
      v8 va;
      if constexpr (F8) {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        const int e = (int) (r / 2), key = e < 4 ? 4 * (int) quad + e : 12 + 4 * (int) quad + e;
        const auto w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*) (tile + T::at(key, t) + 8 * (r & 1)));
        va = from_f8<BF>(u32x2{(uint32_t) w[0], (uint32_t) w[1]});
      } else {
        const int key = 4 * (int) quad + (int) (r / 4), at = 2 * t + (int) (r & 3) / 2, part8 = 8 * (r & 1);
        const s16x4 w0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*) (tile + T::at(key, at) + part8));
        const s16x4 w1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*) (tile + T::at(key + 16, at) + part8));
        va = __builtin_bit_cast(v8, __builtin_shufflevector(w0, w1, 0, 1, 2, 3, 4, 5, 6, 7));
      }
      o[t] = U::mfma16(va, p, o[t]);
    }
  }

  // the waves' results joined: each scaled to the greatest maximum, then summed in the waves' order
  constexpr float kDown = 1.0f / (1 << U::kLift);
  m += (float) U::kLift;
  l = sum_rows(l) * kDown;
  if (quad == 0) ml[wave][0][r] = m, ml[wave][1][r] = l;
  __syncthreads();
  float top = fmaxf(fmaxf(ml[0][0][r], ml[1][0][r]), fmaxf(ml[2][0][r], ml[3][0][r]));
  const float base = finite_max(top), mine = __builtin_amdgcn_exp2f(m - base) * kDown;
  float* out = (float*) lds[wave];
#pragma unroll
  for (int t = 0; t < kDims; t++) *(f32x4*) (out + r * (D + 4) + 16 * t + 4 * quad) = o[t] * mine;
  __syncthreads();
  const float v_scale = F8 && kv.scale ? kv.scale[kv.heads + g] : 1.0f;
  for (uint32_t i = threadIdx.x; i < heads * (D / 4); i += 256) {
    const uint32_t h = i / (D / 4), d = i % (D / 4) * 4;
    f32x4 y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f, top_h = fmaxf(fmaxf(ml[0][0][h], ml[1][0][h]), fmaxf(ml[2][0][h], ml[3][0][h]));
#pragma unroll
    for (int w = 0; w < 4; w++) {
      y += *(const f32x4*) ((const float*) lds[w] + h * (D + 4) + d);
      sum = __builtin_fmaf(ml[w][1][h], __builtin_amdgcn_exp2f(ml[w][0][h] - finite_max(top_h)), sum);
    }
    if (work.n == 1) {
      if (d < a.dim) put4(a, row * a.os + (head0 + h) * a.oh + d, y * (sum == 0.0f ? 0.0f : v_scale / sum));
      if (a.lse && d == 0) a.lse[(uint64_t) row * a.heads + head0 + h] = (top_h + log2f(sum)) * kLn2;
    } else {
      float* to_part = part + ((uint64_t) b * a.heads + head0 + h) * (D + 4);
      *(f32x4*) (to_part + d) = y * v_scale;
      if (d == 0) to_part[D] = top_h, to_part[D + 1] = sum;
    }
  }
}

// the chunks' results of a row and head joined, in the chunks' order (4.4 us after a step of 64 sequences, most of it the
// launch and two dependent loads): a workgroup D / 4 threads of 4 dims in 256 / (D / 4)
// groups, each group every so many chunks, then the groups in order
template <int D>
__global__ __launch_bounds__(256) void join_kernel(Args a, Step st, uint32_t page,
                                                   const uint32_t* __restrict__ cut, const float* __restrict__ part) {
  constexpr uint32_t kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ f32x4 sum4[kGroups][kLanes];
  __shared__ float top_of[kGroups], sum_of[kGroups];
  const uint32_t h = blockIdx.x % a.heads, s = blockIdx.x / a.heads, i = threadIdx.x % kLanes, k = threadIdx.x / kLanes;
  const Seq seq = sequence(st, s, page);
  if (seq.rows < 1) return;
  const uint32_t n = cut[2 * s + 1], row = (uint32_t) (seq.row0 + seq.rows - 1);
  if (n == 1) return;  // (written by its only chunk's workgroup)
  const float* p = part + ((uint64_t) cut[2 * s] * a.heads + h) * (D + 4);
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t c = k; c < n; c += kGroups) {
    const float* pc = p + (uint64_t) c * a.heads * (D + 4);
    const f32x4 o = *(const f32x4*) (pc + 4 * i);
    const float mc = pc[D], lc = pc[D + 1];
    const float top = fmaxf(m, mc), base = finite_max(top), f = __builtin_amdgcn_exp2f(m - base), fc = __builtin_amdgcn_exp2f(mc - base);
    y = y * f + o * fc;
    l = l * f + lc * fc;
    m = top;
  }
  sum4[k][i] = y;
  if (i == 0) top_of[k] = m, sum_of[k] = l;
  __syncthreads();
  if (k) return;
  float top = -__builtin_inff();
#pragma unroll
  for (uint32_t w = 0; w < kGroups; w++) top = fmaxf(top, top_of[w]);
  y = f32x4{0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
#pragma unroll
  for (uint32_t w = 0; w < kGroups; w++) {
    const float f = __builtin_amdgcn_exp2f(top_of[w] - finite_max(top));
    y += sum4[w][i] * f;
    l += sum_of[w] * f;
  }
  if (4 * i < a.dim) put4(a, row * a.os + h * a.oh + 4 * i, y * (l == 0.0f ? 0.0f : 1.0f / l));
  if (a.lse && i == 0) a.lse[(uint64_t) row * a.heads + h] = (top + log2f(l)) * kLn2;
}

template <bool BF, bool F8>
bool run_token(const Args& a, const Kv& k, const Step& st, const Cut& c, uint8_t* workspace, hipStream_t stream) {
  const uint32_t blocks = c.most * k.heads * c.tiles;
  auto* kernel = k.page >= 16 ? (c.dim == 64 ? token_kernel<BF, F8, 64, true> : c.dim == 128 ? token_kernel<BF, F8, 128, true> : token_kernel<BF, F8, 256, true>)
                              : (c.dim == 64 ? token_kernel<BF, F8, 64, false> : c.dim == 128 ? token_kernel<BF, F8, 128, false> : token_kernel<BF, F8, 256, false>);
  uint32_t* cut = c.split ? (uint32_t*) workspace : nullptr;
  float* part = (float*) (workspace + c.head);
  kernel<<<blocks, 256, 0, stream>>>(a, k, st, c.want, c.tiles, cut, part);
  if (hipGetLastError() != hipSuccess) return false;
  if (c.split) {
    auto* join = c.dim == 64 ? join_kernel<64> : c.dim == 128 ? join_kernel<128> : join_kernel<256>;
    join<<<st.n_seq * a.heads, 256, 0, stream>>>(a, st, k.page, cut, part);
  }
  return hipGetLastError() == hipSuccess;
}

// whether the products are taken in bf16
__host__ __device__ inline bool in_bf16(uint32_t kv_type, uint32_t q_type) { return kv_type == OSMOS_BF16 || (kv_type == OSMOS_F8 && q_type == OSMOS_BF16); }

// ---- rows of prompts (osmos_attn_prompt, osmos_attn_chunk) ----
// transposed as above, on v_mfma_f32_32x32x16: a wave holds 32 query rows as columns, a lane one of them (lane % 32) with
// half the keys of a tile (by lane / 32), so that a row's maximum takes one exchange between two lanes and its scaling none, and P^T is the
// second product's B operand as it comes out of the first. a query row is a (token, head) pair of one kv head, the heads
// of a token next to one another: heads that share keys share their loads, a tile of rows covers few tokens (less work
// lost at the causal edge), and a step of few tokens still fills the rows.
// a workgroup is 4 waves of rows over tiles of 32 keys, K and V in LDS twice, pieces of 16 bytes turned by row so that
// neither K's row reads nor V's transposing reads meet a bank twice; one barrier a tile, between the products of one tile (its
// scores', the last tile's outputs') and the next's, so that the waves of a SIMD, of two workgroups, are on the matrix and
// the vector units at different times. measured against it for a prompt of 8192 (32 heads of 128 on 8): 8 waves and tiles of 64
// keys 5 % faster with the second four waves held one phase behind the first, the same without; but prompts of 1 to 2111 tokens
// 11 % slower, chunks over 8-bit pages 22 %, one of 77 tokens 60 %. that prompt takes 583 us, 943 TFLOP/s of the causal half,
// where a library product of 8192 x 8192 x 8192 reaches 1187; the matrix units are busy 45 % of the time and the vector units
// 52 %, and neither reads further ahead, other orders of the phases nor wave priorities changed it.
constexpr int kKeys = 32, kRowWaves = 4;
static_assert(kRows == 32 * kRowWaves);
enum Source { kPacked, kPages, kPagesF8 };

// a row's scores are taken against its running maximum as it was until one is past it by more than this (in powers of two):
// probabilities to 2^8 (in f16, lifted by the rest, to 2^15) cost no accuracy in either type, and most tiles then leave the output
// and the sum unscaled
constexpr int kSlack = 8;

template <int D> struct RowsTile {
  static constexpr int kRow = 2 * D, kBytes = kKeys * kRow;
  static __device__ inline int k_at(int row, int c) { return row * kRow + ((c ^ (D % 128 ? row >> 1 & 7 : row & 15)) * 16); }
  static __device__ inline int v_at(int row, int c) { return row * kRow + ((c ^ (4 * (D % 128 ? row >> 1 & 1 : row & 3))) * 16); }
};

__device__ inline float max_halves(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ inline float sum_halves(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// tile `index` of the step's tiles of kRows query rows: its sequence and its place there. every workgroup finds its own. up to
// 64 sequences (a lane each) in the order of the places, the last places of all sequences first: they see the most keys, and
// what starts late should be short. more sequences from the last to the first, by their running sums
__device__ inline bool find_rows(const Step& st, uint32_t page, uint32_t group, uint32_t index, Seq& seq, uint32_t& tile) {
  const uint32_t lane = threadIdx.x & 63;
  Seq none, q;
  none.row0 = none.rows = none.len = none.end = 0, none.table = st.table;
  auto tiles = [&](const Seq& x) { return (uint32_t) (((uint64_t) (uint32_t) x.rows * group + kRows - 1) / kRows); };
  auto sum = [&](uint32_t x) { return (uint32_t) lane_of((int) wave_scan(x), 63); };
  q = lane < st.n_seq ? sequence(st, lane, page) : none;
  if (st.n_seq <= 64) {
    const uint32_t n = tiles(q);
    if (index >= sum(n)) return false;
    // the greatest place that more than `index` tiles lie at or after
    auto after = [&](uint32_t place) { return sum(n > place ? n - place : 0); };
    uint32_t low = 0, high = 1;
    while (after(high) > index) low = high, high *= 2;
    while (high - low > 1) {
      const uint32_t mid = (low + high) / 2;
      if (after(mid) > index) low = mid;
      else high = mid;
    }
    tile = low;
    uint64_t has = __ballot(n > low);
    for (uint32_t turn = index - after(low + 1); turn; turn--) has &= has - 1;
    seq = lane_of(q, __builtin_ctzll(has));
    return true;
  }
  uint32_t total = 0;
  for (uint32_t s = 0;;) {
    total += sum(tiles(q));
    if ((s += 64) >= st.n_seq) break;
    q = s + lane < st.n_seq ? sequence(st, s + lane, page) : none;
  }
  if (index >= total) return false;
  index = total - 1 - index;
  uint32_t before = 0;
  for (uint32_t s = 0; s < st.n_seq; s += 64) {
    q = s + lane < st.n_seq ? sequence(st, s + lane, page) : none;
    const uint32_t n = tiles(q), x = before + wave_scan(n);
    const uint64_t past = __ballot(x > index);
    if (past) {
      const int at = __builtin_ctzll(past);
      tile = index - ((uint32_t) lane_of((int) x, at) - (uint32_t) lane_of((int) n, at));
      seq = lane_of(q, at);
      return true;
    }
    before = (uint32_t) lane_of((int) x, 63);
  }
  return false;
}

// zeros for the infinities and NaN among 16 bytes of values (e4m3 has NaN alone); whether there were any
template <bool BF, bool F8>
__device__ inline bool take_finite(u32x4& w) {
  constexpr int bits = F8 ? 8 : 16;
  constexpr uint32_t e = F8 ? 0x7Fu : BF ? 0x7F80u : 0x7C00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    uint32_t keep = 0xFFFFFFFFu;
#pragma unroll
    for (int b = 0; b < 32; b += bits)
      if ((w[i] >> b & e) == e) keep &= ~(((1u << bits) - 1) << b), bad = true;
    w[i] &= keep;
  }
  return bad;
}

// the scheduler's order for a block of N scores' products (an LDS read each) and M outputs' (two each), the reads four
// products ahead
template <int N, int M>
__device__ inline void feed() {
  constexpr int kAhead = 4;
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
  for (int i = 0; i < N - kAhead; i++) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
#pragma unroll
  for (int i = 0; i < M; i++) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
}

template <bool BF, int SRC, int D>
__global__ __launch_bounds__(64 * kRowWaves, D > 128 ? 1 : 2) void rows_kernel(Args a, Kv kv, Step st, uint32_t parts,
                                                                               float* __restrict__ part) {
  typedef Unit<BF> U;
  typedef typename U::v8 v8;
  typedef RowsTile<D> T;
  constexpr int kThreads = 64 * kRowWaves, kSteps = D / 16, kDims = D / 32;
  constexpr int kLift = BF ? 0 : U::kLift - kSlack;
  constexpr int kPieces = SRC == kPagesF8 ? kKeys * D / 16 : kKeys * D / 8;  // 16-byte pieces of a tile's keys in memory
  constexpr int kEach = (kPieces + kThreads - 1) / kThreads, kPer = kPieces / kKeys;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][T::kBytes];  // [keys, values][tile & 1]
  typedef std::integral_constant<int, 0> Even;
  typedef std::integral_constant<int, 1> Odd;
  const uint32_t lane = threadIdx.x & 63, wave = (uint32_t) __builtin_amdgcn_readfirstlane((int) threadIdx.x / 64);
  const uint32_t half = lane / 32, col = lane & 31;
  const uint32_t g = blockIdx.x % kv.heads, part_of = blockIdx.x / kv.heads % parts, index = blockIdx.x / kv.heads / parts;
  Seq seq;
  uint32_t tile;
  if (!find_rows(st, SRC == kPacked ? 0 : kv.page, a.group, index, seq, tile)) return;

  // the rows: the workgroup's, the wave's, the lane's, and the positions of their tokens
  const uint32_t all = (uint32_t) seq.rows * a.group, row0 = tile * kRows, last = all - 1 < row0 + kRows - 1 ? all - 1 : row0 + kRows - 1;
  const int base = seq.len - seq.rows;
  const int pos_lo = base + (int) (row0 / a.group), pos_hi = base + (int) (last / a.group);
  const uint32_t wrow = row0 + 32 * wave, wlast = last < wrow + 31 ? last : wrow + 31;
  const int wpos_lo = base + (int) (wrow / a.group), wpos_hi = base + (int) (wlast / a.group);
  const uint32_t row = wrow + col, token = row / a.group, head = g * a.group + row % a.group;
  const bool in = row < all;
  const int pos = base + (int) token;
  const int window = a.window ? (int) a.window : 0x7FFFFFFF;
  int from = a.window && pos_lo >= window ? (pos_lo - window + 1) & ~(kKeys - 1) : 0;
  int to = pos_hi + 1 < seq.end ? pos_hi + 1 : seq.end;
  if (parts > 1 && from < to) {  // (its part of the keys, in whole tiles)
    const int each = ((to - from + kKeys - 1) / kKeys + (int) parts - 1) / (int) parts * kKeys;
    from += (int) part_of * each;
    to = to - from > each ? from + each : to;
  }

  // a thread's 16-byte pieces of a tile: of rows key_row(i). stage s writes the keys of tile s + 1 and the values of tile s
  // into LDS, loaded into registers a tile's time before; page ids are loaded one stage ahead of that. past the last tile
  // the last is loaded and written again, which no one reads: the products' phase has no conditions in it
  const uint32_t size = SRC == kPagesF8 ? 1 : 2, dim_bytes = a.dim * size, shift = SRC == kPacked ? 0 : 31 - __builtin_clz(kv.page);
  const uint64_t page_bytes = (uint64_t) kv.heads * kv.page * dim_bytes, head_at = (uint64_t) g * kv.page * dim_bytes;
  const int n = from < to ? (to - from + kKeys - 1) / kKeys : 0;
  u32x4 kr[kEach], vr[kEach];
  int kid[kEach], vid[kEach], live_id = 0;
  uint32_t live_old = 0, live = 0, live_new = 0;  // of tiles s - 1, s and s + 1: the keys that are there, a bit each
  auto key_row = [&](int i) __attribute__((always_inline)) { return (int) ((threadIdx.x + i * kThreads) / kPer) & (kKeys - 1); };
  auto piece = [&](int i) __attribute__((always_inline)) { return (threadIdx.x + i * kThreads) % kPer; };
  auto start = [&](int t) __attribute__((always_inline)) { return from + (t < n ? t : n - 1) * kKeys; };
  auto clamp_key = [&](int j) __attribute__((always_inline)) { return j < to ? j : to - 1; };
  auto ids = [&](int t) __attribute__((always_inline)) {
    if constexpr (SRC != kPacked) {
#pragma unroll
      for (int i = 0; i < kEach; i++) vid[i] = kid[i], kid[i] = gload<int>(seq.table + ((uint32_t) clamp_key(start(t) + key_row(i)) >> shift));
      live_id = gload<int>(seq.table + ((uint32_t) clamp_key(start(t) + (int) (lane & (kKeys - 1))) >> shift));
    }
  };
  // packed rows: where tiles of keys and of values lie, the next of each to be loaded
  const uint8_t *kplace = kv.k + ((uint64_t) (seq.row0 + from) * kv.ks + g * kv.kh) * 2, *vplace = kv.v + ((uint64_t) (seq.row0 + from) * kv.vs + g * kv.vh) * 2;
  auto load = [&](int t, const uint8_t*& plane, uint32_t stride, const int (&id)[kEach], u32x4 (&to_regs)[kEach]) __attribute__((always_inline)) {
    const int j0 = start(t);
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      const uint32_t d = piece(i) * 16 < dim_bytes ? piece(i) * 16 : 0;
      if constexpr (SRC == kPacked) {  // (a place that is the wave's, and the lane's from there)
        to_regs[i] = gload<u32x4>(plane + ((uint32_t) (clamp_key(j0 + key_row(i)) - j0) * (stride * 2) + d));
      } else {
        const uint32_t page = (uint32_t) id[i] < kv.pages ? (uint32_t) id[i] : 0u, slot = (uint32_t) clamp_key(j0 + key_row(i)) & (kv.page - 1);
        to_regs[i] = gload<u32x4>(plane + (page * page_bytes + head_at + slot * dim_bytes + d));
      }
    }
    if (SRC == kPacked && t + 1 < n) plane += (uint64_t) stride * (2 * kKeys);
  };
  if constexpr (SRC != kPacked) kplace = kv.k, vplace = kv.v;
  auto there = [&](int t) __attribute__((always_inline)) {
    return (uint32_t) __ballot(start(t) + (int) (lane & (kKeys - 1)) < to && (SRC == kPacked || (uint32_t) live_id < kv.pages));
  };
  auto load_stage = [&](int s) __attribute__((always_inline)) {
    live_old = live, live = live_new, live_new = there(s + 1);
    load(s + 1, kplace, (uint32_t) kv.ks, kid, kr);
    load(s, vplace, (uint32_t) kv.vs, vid, vr);
    ids(s + 2);
  };
  // what must not reach LDS: keys' pieces past the dims (q is zeros there, but 0 times an infinity would be NaN); values of
  // keys that are not there (masked, they have no influence); and in a tile that some of the rows see in part infinities and
  // NaN, as 0 times them would reach the rows that do not see them: those that do get them at the end
  auto partial = [&](int j0) __attribute__((always_inline)) { return j0 + kKeys - 1 > pos_lo || j0 <= pos_hi - window; };
  bool bad = false;
  auto mend_stage = [&](int s) __attribute__((always_inline)) {
    if (a.dim < D) {
      asm volatile("");  // (a branch: selects would wait for the loads here, in every tile)
#pragma unroll
      for (int i = 0; i < kEach; i++)
        if (piece(i) * 16 >= dim_bytes) kr[i] = u32x4{0, 0, 0, 0};
    }
    const bool part = partial(start(s));
    if (part || live != ~0u) {
      asm volatile("");
#pragma unroll
      for (int i = 0; i < kEach; i++) {
        if (!(live >> key_row(i) & 1)) vr[i] = u32x4{0, 0, 0, 0};
        if (part && take_finite<BF, SRC == kPagesF8>(vr[i])) bad = true;
      }
    }
  };
  auto write = [&](uint8_t* to_tile, bool values, const u32x4 (&regs)[kEach]) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kEach; i++) {
      if (kPieces % kThreads && threadIdx.x + i * kThreads >= kPieces) break;
      const int r = key_row(i), c = (int) piece(i);
      if constexpr (SRC == kPagesF8) {
#pragma unroll
        for (int w = 0; w < 2; w++)
          *(u32x4*) (to_tile + (values ? T::v_at(r, 2 * c + w) : T::k_at(r, 2 * c + w))) = __builtin_bit_cast(u32x4, from_f8<BF>(u32x2{regs[i][2 * w], regs[i][2 * w + 1]}));
      } else {
        *(u32x4*) (to_tile + (values ? T::v_at(r, c) : T::k_at(r, c))) = regs[i];
      }
    }
  };
  // the end of a tile's products: LDS writes done and seen; loads from memory stay in flight
  auto meet = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  if (n) {
    ids(0);
    live_new = there(0);
    load(0, kplace, (uint32_t) kv.ks, kid, kr);
    ids(1);
  }
  v8 q[kSteps];
  const float scale = a.scale * (SRC == kPagesF8 && kv.scale ? kv.scale[g] : 1.0f), unit = unit_of(scale);
  load_q<BF, kSteps>(a, (uint64_t) seq.row0 + (in ? token : 0), in ? head : 0, in, scale,
                     [&](int i) { return (uint32_t) (16 * i + 8 * half); }, q);
  f32x16 o[kDims], x;
#pragma unroll
  for (int i = 0; i < kDims; i++) o[i] = f32x16{};
  v8 p[2];
  float m = -__builtin_inff(), l = 0.0f;

  // a lane's places in a tile's keys and values: all of them by one exclusive or and one addition from the first (D a power
  // of two), made anew for each tile, as there are no registers to keep them in
  const int vrow = (int) (4 * half + (lane & 15) / 4), vdims = (int) (16 * (lane >> 4 & 1) + 4 * (lane & 3));
  const uint32_t kfirst = (uint32_t) T::k_at((int) col, (int) half), vfirst = (uint32_t) (T::v_at(vrow, vdims / 8) + vdims % 8 * 2);
  auto scores = [&](const uint8_t* kt) __attribute__((always_inline)) {
    uint32_t at0 = kfirst;
    asm volatile("" : "+v"(at0));
    x = f32x16{};
#pragma unroll
    for (int i = 0; i < kSteps; i++) {
      const uint32_t at = (D & (D - 1)) == 0 ? at0 ^ (uint32_t) (32 * i) : (uint32_t) T::k_at((int) col, 2 * i + (int) half);
      x = U::mfma32(*(const v8*) (kt + at), q[i], x);
    }
  };
  auto outputs = [&](const uint8_t* vt) __attribute__((always_inline)) {
    // V^T's columns of keys 16 u + 4 half + 0 .. 3 and 8 more on, as P^T's lanes hold them
    uint32_t at0 = vfirst;
    asm volatile("" : "+v"(at0));
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int i = 0; i < kDims; i++) {
        const uint32_t at = (D & (D - 1)) == 0 ? (at0 ^ (uint32_t) (64 * i)) + (uint32_t) (16 * u * T::kRow) : (uint32_t) (T::v_at(16 * u + vrow, 4 * i + vdims / 8) + vdims % 8 * 2);
        const s16x4 w0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*) (vt + at));
        const s16x4 w1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*) (vt + at + 8 * T::kRow));
        o[i] = U::mfma32(__builtin_bit_cast(v8, __builtin_shufflevector(w0, w1, 0, 1, 2, 3, 4, 5, 6, 7)), p[u], o[i]);
      }
  };
  auto softmax = [&](int t) __attribute__((always_inline)) {
    const int j0 = start(t);
    if (live_old != ~0u || j0 + kKeys - 1 > wpos_lo || (a.window && j0 <= wpos_hi - window)) {
      // the row's keys are lo + 1 .. hi of the tile (less the half's 4, so that the lane's keys are constants)
      const int hi = pos - j0 - 4 * (int) half, lo = a.window && pos >= window ? pos - window - j0 - 4 * (int) half : -5;
      const uint32_t mine = live_old >> (4 * half);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        const int key = 8 * (i / 4) + i % 4;
        if (key > hi || key <= lo || !(mine >> key & 1)) x[i] = -__builtin_inff();
      }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, x[i]);
    top = __builtin_fmaf(max_halves(top), unit, -(float) kLift);
    if (__any(top > m + (float) kSlack)) {
      const float next = fmaxf(m, top), fade = __builtin_amdgcn_exp2f(m - finite_max(next));
      m = next;
      l *= fade;
#pragma unroll
      for (int i = 0; i < kDims; i++) o[i] *= fade;
    }
    const float sub = finite_max(m);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], unit, -sub));
      sum = i ? sum + e : e;
      p[i / 8][i % 8] = (typename U::e) e;
    }
    l += sum;
  };
  // the products' phase after tile t's softmax: the next tile's scores, tile t's outputs, the next stage
  auto products = [&](int t, auto buf) __attribute__((always_inline)) {
    constexpr int b = decltype(buf)::value;
    scores(lds[0][1 - b]);
    outputs(lds[1][b]);
    feed<kSteps, 2 * kDims>();
    mend_stage(t + 1);
    write(lds[0][b], false, kr);
    write(lds[1][1 - b], true, vr);
    load_stage(t + 2);
  };

  if (n) {
    if (a.dim < D) {
#pragma unroll
      for (int i = 0; i < kEach; i++)
        if (piece(i) * 16 >= dim_bytes) kr[i] = u32x4{0, 0, 0, 0};
    }
    write(lds[0][0], false, kr);
    load_stage(0);
    meet();
    mend_stage(0);
    scores(lds[0][0]);
    write(lds[0][1], false, kr);
    write(lds[1][0], true, vr);
    load_stage(1);
    meet();
    int t = 0;
    for (; t + 2 < n; t += 2) {
      softmax(t);
      products(t, Even());
      meet();
      softmax(t + 1);
      products(t + 1, Odd());
      meet();
    }
    softmax(t);
    if (t + 1 < n) {
      products(t, Even());
      meet();
      softmax(++t);
    }
    outputs(lds[1][t & 1]);
  }

  if (__syncthreads_or(bad)) {
    // seldom: the infinities and NaN left out above, added to the rows that see their keys
    for (int t = from; t < to; t += kKeys)
      if (partial(t))
        for (int j = t; j < (t + kKeys < to ? t + kKeys : to); j++) {
          uint64_t at;
          if constexpr (SRC == kPacked) {
            at = ((uint64_t) (seq.row0 + j) * kv.vs + g * kv.vh) * 2;
          } else {
            const uint32_t page = (uint32_t) seq.table[(uint32_t) j >> shift];
            if (page >= kv.pages) continue;
            at = page * page_bytes + head_at + ((uint32_t) j & (kv.page - 1)) * dim_bytes;
          }
          if (j > pos || j <= pos - window) continue;
#pragma unroll
          for (int i = 0; i < kDims; i++)
#pragma unroll
            for (int n = 0; n < 4; n++) {
              const uint32_t d = 32 * i + 8 * n + 4 * half;
              if (d >= a.dim) continue;
              f32x4 w;
              if constexpr (SRC == kPagesF8) {
                const uint32_t x = gload<uint32_t>(kv.v + at + d);
                const auto low = U::f8_low(x), high = U::f8_high(x);
                w = f32x4{(float) low[0], (float) low[1], (float) high[0], (float) high[1]};
              } else {
                const typename U::v4 x = gload<typename U::v4>(kv.v + at + d * 2);
                w = f32x4{(float) x[0], (float) x[1], (float) x[2], (float) x[3]};
              }
#pragma unroll
              for (int e = 0; e < 4; e++)
                if (!(fabsf(w[e]) < __builtin_inff())) o[i][4 * n + e] += w[e];
            }
        }
  }
  if (!in) return;
  constexpr float kDown = 1.0f / (1 << kLift);
  const float v_scale = (SRC == kPagesF8 && kv.scale ? kv.scale[kv.heads + g] : 1.0f) * kDown;
  m += (float) kLift;
  l = sum_halves(l) * kDown;
  if (parts > 1) {
    float* at = part + ((uint64_t) blockIdx.x * kRows + (row - row0)) * (D + 4);
#pragma unroll
    for (int i = 0; i < kDims; i++)
#pragma unroll
      for (int n = 0; n < 4; n++)
        *(f32x4*) (at + 32 * i + 8 * n + 4 * half) = f32x4{o[i][4 * n], o[i][4 * n + 1], o[i][4 * n + 2], o[i][4 * n + 3]} * v_scale;
    if (half == 0) at[D] = m, at[D + 1] = l;
    return;
  }
  const float inv = l == 0.0f ? 0.0f : v_scale / l;
  const uint64_t at = ((uint64_t) seq.row0 + token) * a.os + head * a.oh;
#pragma unroll
  for (int i = 0; i < kDims; i++)
#pragma unroll
    for (int n = 0; n < 4; n++) {
      const uint32_t d = 32 * i + 8 * n + 4 * half;
      if (d < a.dim) put4(a, at + d, f32x4{o[i][4 * n], o[i][4 * n + 1], o[i][4 * n + 2], o[i][4 * n + 3]} * inv);
    }
  if (a.lse && half == 0) a.lse[((uint64_t) seq.row0 + token) * a.heads + head] = (m + log2f(l)) * kLn2;
}

// the parts' results of each row joined, in the parts' order: D / 4 lanes (a power of two of them) a row
template <int D>
__global__ __launch_bounds__(256) void rows_join_kernel(Args a, Step st, uint32_t page, uint32_t kv_heads, uint32_t parts,
                                                        const float* __restrict__ part) {
  constexpr uint32_t kLanes = D <= 64 ? 16 : D <= 128 ? 32 : 64, kEach = 256 / kLanes;
  uint32_t b = blockIdx.x;
  const uint32_t piece = b % (kRows / kEach);
  b /= kRows / kEach;
  const uint32_t g = b % kv_heads, index = b / kv_heads;
  Seq seq;
  uint32_t tile;
  if (!find_rows(st, page, a.group, index, seq, tile)) return;
  const uint32_t r = piece * kEach + threadIdx.x / kLanes, d = threadIdx.x % kLanes * 4, row = tile * kRows + r;
  if (row >= (uint32_t) seq.rows * a.group || d >= a.dim) return;
  const float* p = part + (((uint64_t) index * parts * kv_heads + g) * kRows + r) * (D + 4);
  const uint64_t step = (uint64_t) kv_heads * kRows * (D + 4);
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (uint32_t c = 0; c < parts; c++) {
    const f32x4 o = *(const f32x4*) (p + c * step + d);
    const float mc = p[c * step + D], lc = p[c * step + D + 1];
    const float top = fmaxf(m, mc), base = finite_max(top), f = __builtin_amdgcn_exp2f(m - base), fc = __builtin_amdgcn_exp2f(mc - base);
    y = y * f + o * fc;
    l = l * f + lc * fc;
    m = top;
  }
  const uint32_t token = (uint32_t) seq.row0 + row / a.group, head = g * a.group + row % a.group;
  put4(a, (uint64_t) token * a.os + head * a.oh + d, y * (l == 0.0f ? 0.0f : 1.0f / l));
  if (a.lse && d == 0) a.lse[(uint64_t) token * a.heads + head] = (m + log2f(l)) * kLn2;
}

template <bool BF, int SRC>
bool run_rows(const Args& a, const Kv& k, const OsmosKvStep* step, const RowsCut& c, float* part, hipStream_t stream) {
  const Step st = kv::step_of(step);
  auto* kernel = c.dim == 64 ? rows_kernel<BF, SRC, 64> : c.dim == 128 ? rows_kernel<BF, SRC, 128> : c.dim == 192 ? rows_kernel<BF, SRC, 192> : rows_kernel<BF, SRC, 256>;
  kernel<<<(uint32_t) (c.tiles * k.heads * c.parts), 64 * kRowWaves, 0, stream>>>(a, k, st, c.parts, part);
  if (hipGetLastError() != hipSuccess) return false;
  if (c.parts > 1) {
    const uint32_t pieces = kRows / (c.dim == 64 ? 16 : c.dim == 128 ? 8 : 4);
    auto* join = c.dim == 64 ? rows_join_kernel<64> : c.dim == 128 ? rows_join_kernel<128> : c.dim == 192 ? rows_join_kernel<192> : rows_join_kernel<256>;
    join<<<(uint32_t) (c.tiles * k.heads * pieces), 256, 0, stream>>>(a, st, SRC == kPacked ? 0 : k.page, k.heads, c.parts, part);
  }
  return hipGetLastError() == hipSuccess;
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

}  // namespace attn
}  // namespace osm

using namespace osm;

extern "C" OSM_API uint64_t osmos_attn_workspace(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim,
                                                 const OsmosKvStep* step) {
  if (!a || !a->heads || !kv_heads || a->heads % kv_heads || !dim || dim > OSMOS_ATTN_MAX_DIM || !step) return 0;
  if (!step->n_seq || !step->n_tok) return 0;
  const uint64_t rows = attn::rows_bytes(attn::rows_cut(a, kv_heads, dim, step), kv_heads);
  const uint64_t token = step->max_tok == 1 && step->len ? attn::token_bytes(a, attn::cut_of(a, kv_heads, dim, step)) : 0;
  return rows > token ? rows : token;
}

extern "C" OSM_API bool osmos_attn_prompt(const OsmosAttn* a, const OsmosKvRows* r, const OsmosKvStep* step,
                                          void* workspace, uint64_t workspace_bytes, void* stream) {
  if (!attn::prompt_ok(a, r, step, workspace, workspace_bytes)) return false;
  const attn::Kv k{(const uint8_t*) r->k, (const uint8_t*) r->v, r->k_stride, r->k_head, r->v_stride, r->v_head, r->type,
                   0, 0, r->heads, nullptr};
  auto* run = r->type == OSMOS_BF16 ? attn::run_rows<true, attn::kPacked> : attn::run_rows<false, attn::kPacked>;
  return run(attn::args_of(a, r->heads, r->dim), k, step, attn::rows_cut(a, r->heads, r->dim, step), (float*) workspace,
             (hipStream_t) stream);
}

extern "C" OSM_API bool osmos_attn_chunk(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step,
                                         void* workspace, uint64_t workspace_bytes, void* stream) {
  if (!attn::chunk_ok(a, kv, layer, step, workspace, workspace_bytes)) return false;
  const bool bf = attn::in_bf16(kv->type, a->q_type), f8 = kv->type == OSMOS_F8;
  auto* run = bf ? (f8 ? attn::run_rows<true, attn::kPagesF8> : attn::run_rows<true, attn::kPages>)
                 : (f8 ? attn::run_rows<false, attn::kPagesF8> : attn::run_rows<false, attn::kPages>);
  return run(attn::args_of(a, kv->heads, kv->dim), attn::pages_of(kv, layer), step, attn::rows_cut(a, kv->heads, kv->dim, step),
             (float*) workspace, (hipStream_t) stream);
}

extern "C" OSM_API bool osmos_attn_token(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step,
                                         void* workspace, uint64_t workspace_bytes, void* stream) {
  if (!attn::token_ok(a, kv, layer, step, workspace, workspace_bytes)) return false;
  const bool bf = attn::in_bf16(kv->type, a->q_type), f8 = kv->type == OSMOS_F8;
  auto* run = bf ? (f8 ? attn::run_token<true, true> : attn::run_token<true, false>)
                 : (f8 ? attn::run_token<false, true> : attn::run_token<false, false>);
  return run(attn::args_of(a, kv->heads, kv->dim), attn::pages_of(kv, layer), kv::step_of(step),
             attn::cut_of(a, kv->heads, kv->dim, step), (uint8_t*) workspace, (hipStream_t) stream);
}
