// libosmos MI355X - how the attention's launches are cut (attn.hip): plain arithmetic, so that the host can check every cut that a
// step's lengths can make.
#pragma once
#include <stdint.h>

#include "../../include/osmos_attn.h"

namespace osm {
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

// how a token step is launched: the chunks that the sequences are cut into for each kv head and 16 of its query heads (the
// chip holds 512 of their workgroups; 512 / 768 / 1024 / 2048 wanted measured 99 / 100 / 106 / 112 us for one sequence of 131072 and
// 44 / 45 / 43 / 50 for 64 of 1 to 8192; chunks of at least 256 / 384 / 512 keys 9.3 / 6.4 / 6.4 us for one of 333, which
// then needs no join, and 20 / 17 / 17.5 for 24 wide 8-bit ones), and the workspace: where each sequence's chunks begin and
// how many they are, then the chunks' results
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

}  // namespace attn
}  // namespace osm
