// what the paged cache's and the attention's entry points decide on the host (attnhost.h), as a shared library for the tests
#include "../libosmos_amd/csrc/attnhost.h"

using namespace osm;

extern "C" {
uint32_t host_chunk_keys(uint32_t total, uint32_t want) { return attn::chunk_keys(total, want); }
uint32_t host_chunks_of(int k, uint32_t chunk) { return attn::chunks_of(k, chunk); }
void host_cut(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim, const OsmosKvStep* st, uint32_t* want, uint32_t* most,
              uint32_t* split) {
  const attn::Cut c = attn::cut_of(a, kv_heads, dim, st);
  *want = c.want, *most = c.most, *split = c.split;
}

bool host_append(const OsmosKv* kv, uint32_t layer, const OsmosKvStep* st, uint32_t type, const void* k, uint64_t ks,
                 const void* v, uint64_t vs) {
  return kv::append_ok(kv, layer, st, type, k, ks, v, vs);
}
bool host_requests(const OsmosKv* kv, const OsmosKvPool* p, const int32_t* a, const int32_t* b, uint32_t n) {
  return kv::requests_ok(kv, p, a, b, n);
}
bool host_pool(const OsmosKv* kv, const OsmosKvPool* p) { return kv::pool_ok(kv, p); }
bool host_copy(const OsmosKv* kv, const int32_t* a, const int32_t* b, uint32_t n) { return kv::copy_ok(kv, a, b, n); }
bool host_prompt(const OsmosAttn* a, const OsmosKvRows* r, const OsmosKvStep* st, const void* ws, uint64_t bytes) {
  return attn::prompt_ok(a, r, st, ws, bytes);
}
bool host_chunk(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* st, const void* ws, uint64_t bytes) {
  return attn::chunk_ok(a, kv, layer, st, ws, bytes);
}
bool host_token(const OsmosAttn* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* st, const void* ws, uint64_t bytes) {
  return attn::token_ok(a, kv, layer, st, ws, bytes);
}
}
