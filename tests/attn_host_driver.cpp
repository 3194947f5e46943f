// a token step's cut (attnhost.h), for tests of the host: built as a shared library
#include "../libosmos_amd/csrc/attnhost.h"

extern "C" {
uint32_t host_chunk_keys(uint32_t total, uint32_t want) { return osm::attn::chunk_keys(total, want); }
uint32_t host_chunks_of(int k, uint32_t chunk) { return osm::attn::chunks_of(k, chunk); }
void host_cut(const OsmosAttn* a, uint32_t kv_heads, uint32_t dim, const OsmosKvStep* st, uint32_t* want, uint32_t* most,
              uint32_t* split) {
  const osm::attn::Cut c = osm::attn::cut_of(a, kv_heads, dim, st);
  *want = c.want, *most = c.most, *split = c.split;
}
}
