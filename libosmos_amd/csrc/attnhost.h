// libosmos MI355X - what the paged cache's and the attention's entry points (kv.hip, attn.hip) decide before they queue anything:
// what they refuse, and how their launches are cut. plain C++, so that the host can check it by itself: a call that a lost check
// lets through cannot be told from a refused one where there is no GPU.
#pragma once
#include <stdint.h>

#include "../../include/osmos_attn.h"

namespace osm {
namespace kv {

constexpr uint32_t size_of(uint32_t type) { return type == OSMOS_F32 ? 4 : type == OSMOS_F8 ? 1 : 2; }
inline bool row_type(uint32_t t) { return t == OSMOS_F32 || t == OSMOS_F16 || t == OSMOS_BF16; }

inline bool shape_ok(const OsmosKv* kv) {
  if (!kv || (kv->type != OSMOS_F16 && kv->type != OSMOS_BF16 && kv->type != OSMOS_F8)) return false;
  if (!kv->layers || kv->layers > 4096 || !kv->pages || kv->pages > 0x7FFFFFF0u || !kv->heads || kv->heads > 4096) return false;
  if (!kv->page || kv->page > OSMOS_KV_MAX_PAGE || (kv->page & (kv->page - 1))) return false;
  return kv->dim && kv->dim <= OSMOS_ATTN_MAX_DIM && kv->dim % 16 == 0 &&
         (uint64_t) kv->heads * kv->page * kv->dim <= OSMOS_KV_MAX_PAGE_VALUES;
}
inline uint64_t page_bytes(const OsmosKv* kv) { return (uint64_t) kv->heads * kv->page * kv->dim * size_of(kv->type); }
inline uint64_t plane_bytes(const OsmosKv* kv) { return page_bytes(kv) * kv->pages; }
inline bool cache_ok(const OsmosKv* kv) {
  return shape_ok(kv) && kv->data && (uintptr_t) kv->data % 16 == 0 && (kv->type == OSMOS_F8 || !kv->scale);
}
inline bool step_ok(const OsmosKvStep* st, bool paged) {
  if (!st || !st->start || !st->n_seq || st->n_seq > 0x100000u || !st->n_tok || st->n_tok > 0x7FFFFFFFu || !st->max_tok ||
      st->max_tok > 0x7FFFFFFFu)
    return false;
  if (!paged) return true;
  return st->len && st->table && st->table_stride && st->seqs && (st->seq || st->n_seq <= st->seqs) && st->max_len &&
         st->max_len <= 0x7FFF0000u;
}
inline bool append_ok(const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step, uint32_t type, const void* k,
                      uint64_t k_stride, const void* v, uint64_t v_stride) {
  if (!cache_ok(kv) || layer >= kv->layers || !step_ok(step, true) || !k || !v || !row_type(type)) return false;
  const uint64_t row = (uint64_t) kv->heads * kv->dim, size = size_of(type);
  if ((uintptr_t) k % 16 || (uintptr_t) v % 16 || k_stride * size % 16 || v_stride * size % 16) return false;
  return step->n_tok == 1 || (k_stride >= row && v_stride >= row);
}

// a pool's scratch: three lists of whole 16-page pieces, then the copy list and the counts
inline uint64_t list_ints(const OsmosKv* kv) { return (kv->pages + 15ull) / 16 * 16; }
inline bool pool_ok(const OsmosKv* kv, const OsmosKvPool* p) {
  return cache_ok(kv) && p && p->ref && (uintptr_t) p->ref % 16 == 0 && p->len && p->table && p->scratch &&
         (uintptr_t) p->scratch % 16 == 0 && p->seqs && p->seqs <= 0x7FFFFFFFu && p->table_stride;
}
inline bool requests_ok(const OsmosKv* kv, const OsmosKvPool* p, const int32_t* a, const int32_t* b, uint32_t n) {
  return pool_ok(kv, p) && a && b && n && n <= OSMOS_KV_MAX_REQUESTS;
}
inline bool copy_ok(const OsmosKv* kv, const int32_t* from, const int32_t* to, uint32_t n) { return cache_ok(kv) && from && to && n; }

}  // namespace kv

namespace attn {

// a token step's keys are cut into chunks of one length, so that `want` of them hold all its `total` tiles of 32 (at least kLeast
// keys each, whole 128s: a tile for each wave). a sequence has under 2^31 - 128 keys: where the even share would pass that (2^26
// tiles a chunk), every sequence is one chunk
constexpr uint32_t kLeast = 384;
constexpr uint32_t chunk_keys(uint32_t total, uint32_t want) {
  const uint32_t share = total / want, even = (share < (1u << 26) - 5 ? share : (1u << 26) - 5) + 1;
  return even * 32 <= kLeast ? kLeast : (even + 3) / 4 * 128;
}
// the chunks of a sequence of k keys
constexpr uint32_t chunks_of(int k, uint32_t chunk) { return (uint32_t) k <= chunk ? 1 : ((uint32_t) k + chunk - 1) / chunk; }

// how a token step is launched: the chunks that the sequences are cut into for each kv head and 16 of its query heads, and the
// workspace: where each sequence's chunks begin and how many they are, then the chunks' results. 512 workgroups are what the
// chip holds of the instances for 16-bit heads of 128 and 8-bit ones of 256, two a compute unit (16-bit 256: one, 8-bit 128:
// three, heads of 64: four or five). 512 / 768 / 1024 / 2048 wanted measured 99 / 100 / 106 / 112 us for one sequence of 131072
// and 44 / 45 / 43 / 50 for 64 of 1 to 8192, both 16-bit heads of 128; the other instances take the same number unmeasured. chunks
// of at least 256 / 384 / 512 keys 9.3 / 6.4 / 6.4 us for one of 333, which then needs no join, and 20 / 17 / 17.5 for 24 8-bit
// ones of heads of 256
constexpr uint32_t kWant = 512;
struct Cut {
  uint32_t want, most, tiles, dim;  // most: chunks there can be
  bool split;                       // whether a sequence can have more than one
  uint64_t head;                    // the workspace's bytes before the results
};
inline Cut cut_of(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim, const OsmosKvStep* st) {
  Cut c;
  c.tiles = (a->heads / kv_heads + 15) / 16;
  c.dim = dim <= 64 ? 64 : dim <= 128 ? 128 : 256;
  c.want = kWant / (kv_heads * c.tiles) ? kWant / (kv_heads * c.tiles) : 1;
  const uint64_t keys = a->window && a->window + 31ull < st->max_len ? a->window + 31ull : st->max_len;
  c.split = keys > kLeast;
  const uint64_t each = st->n_seq * ((keys + kLeast - 1) / kLeast), even = (uint64_t) c.want + st->n_seq;
  c.most = (uint32_t) (each < even ? each : even);
  c.head = (st->n_seq * 8ull + 255) / 256 * 256;
  return c;
}
inline uint64_t token_bytes(const OsmosAttn* a, const Cut& c) {
  return c.split ? c.head + (uint64_t) c.most * a->heads * (c.dim + 4) * 4 : 0;
}

constexpr int kRows = 128;  // query rows a workgroup of rows_kernel

// how the rows are launched: tiles there can be, and the parts that each tile's keys are cut into: one, but where the tiles
// leave compute units without work and the keys are many (a part of 256 keys or more, so that it costs more than its join).
// 923 rows of 24 heads over 7109 tokens of 8-bit pages (184 tiles at most): whole 175 us, for 512 / 768 / 1024 / 1536 / 2048
// workgroups 131 / 114 / 102 / 96 / 105; other head sizes and page types take the same number unmeasured
constexpr uint64_t kFull = 1536, kLeastPart = 256;
struct RowsCut {
  uint64_t tiles;
  uint32_t parts, dim;
};
inline RowsCut rows_cut(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim, const OsmosKvStep* st) {
  RowsCut c;
  c.tiles = (uint64_t) st->n_tok * (a->heads / kv_heads) / kRows + (st->n_seq < st->n_tok ? st->n_seq : st->n_tok);
  const uint64_t blocks = c.tiles * kv_heads, longest = st->len ? st->max_len : st->max_tok;
  uint64_t keys = longest;
  if (a->window && a->window + (uint64_t) kRows + 31 < keys) keys = a->window + (uint64_t) kRows + 31;
  uint64_t parts = blocks ? kFull / blocks : 1;
  if (parts > keys / kLeastPart) parts = keys / kLeastPart;
  c.parts = (uint32_t) (parts < 1 ? 1 : parts > 64 ? 64 : parts);
  c.dim = dim <= 64 ? 64 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;
  return c;
}
inline uint64_t rows_bytes(const RowsCut& c, uint32_t kv_heads) {
  return c.parts > 1 ? c.tiles * kv_heads * c.parts * kRows * (c.dim + 4) * 4 : 0;
}

// what the calls refuse
inline bool room_ok(uint64_t need, const void* workspace, uint64_t bytes) {
  return !need || (workspace && (uintptr_t) workspace % 256 == 0 && bytes >= need);
}
inline bool stride_ok(uint64_t stride, uint32_t type) { return stride * kv::size_of(type) % 16 == 0; }
inline bool args_ok(const OsmosAttn* a, uint32_t kv_heads) {
  if (!a || !a->q || !a->out || (uintptr_t) a->q % 16 || (uintptr_t) a->out % 16) return false;
  if (!kv::row_type(a->q_type) || !kv::row_type(a->out_type) || !a->heads || a->heads > 4096 || a->heads % kv_heads) return false;
  if (!stride_ok(a->q_stride, a->q_type) || !stride_ok(a->q_head, a->q_type) || !stride_ok(a->out_stride, a->out_type) ||
      !stride_ok(a->out_head, a->out_type))
    return false;
  return a->window <= 0x7FFFFFFFu && a->scale == a->scale;
}
inline bool rows_fit(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim, const OsmosKvStep* step, const void* workspace,
                     uint64_t bytes) {
  const RowsCut c = rows_cut(a, kv_heads, dim, step);
  return c.tiles * kv_heads * c.parts <= 0x7FFFFFFFull && (uint64_t) step->n_tok * (a->heads / kv_heads) <= 0x7FFFFFFFull &&
         room_ok(rows_bytes(c, kv_heads), workspace, bytes);
}
inline bool prompt_ok(const OsmosAttn* a, const OsmosKvRows* r, const OsmosKvStep* step, const void* workspace, uint64_t bytes) {
  if (!r || !r->k || !r->v || !r->heads || r->heads > 4096 || (r->type != OSMOS_F16 && r->type != OSMOS_BF16)) return false;
  if (!r->dim || r->dim > OSMOS_ATTN_MAX_DIM || r->dim % 16 || (uintptr_t) r->k % 16 || (uintptr_t) r->v % 16) return false;
  if (r->k_stride % 8 || r->k_head % 8 || r->v_stride % 8 || r->v_head % 8) return false;
  if (r->k_stride > OSMOS_ATTN_MAX_STRIDE || r->v_stride > OSMOS_ATTN_MAX_STRIDE) return false;
  return args_ok(a, r->heads) && kv::step_ok(step, false) && rows_fit(a, r->heads, r->dim, step, workspace, bytes);
}
inline bool paged_ok(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step) {
  return kv::cache_ok(kv) && layer < kv->layers && args_ok(a, kv->heads) && kv::step_ok(step, true);
}
inline bool chunk_ok(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step, const void* workspace,
                     uint64_t bytes) {
  return paged_ok(a, kv, layer, step) && rows_fit(a, kv->heads, kv->dim, step, workspace, bytes);
}
inline bool token_ok(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* step, const void* workspace,
                     uint64_t bytes) {
  if (!paged_ok(a, kv, layer, step) || step->max_tok != 1) return false;
  // (a step's tiles are counted in 32 bits)
  const uint64_t room = (uint64_t) step->table_stride * kv->page, longest = room < step->max_len ? room : step->max_len;
  if (step->n_seq * (longest / 32 + 1) > 0xFFFFFFFFull) return false;
  const Cut c = cut_of(a, kv->heads, kv->dim, step);
  return (uint64_t) c.most * kv->heads * c.tiles <= 0x7FFFFFFFull && (uint64_t) step->n_seq * a->heads <= 0x7FFFFFFFull &&
         room_ok(token_bytes(a, c), workspace, bytes);
}

}  // namespace attn
}  // namespace osm
