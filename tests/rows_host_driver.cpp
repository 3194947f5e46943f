// what include/osmos_rows.h's entry points decide on the host (rowshost.h), as a shared library for the tests
#include "../libosmos_amd/csrc/rowshost.h"

using namespace osm;

extern "C" {
bool host_norm(const OsmosNorm* a) { return rows::norm_ok(a); }
bool host_rope(const OsmosRope* a) { return rows::rope_ok(a, false); }
bool host_rope_append(const OsmosRope* a, const OsmosKv* kv, uint32_t layer, const OsmosKvStep* st, const void* v, uint64_t vs, uint64_t vh) {
  return rows::rope_append_ok(a, kv, layer, st, v, vs, vh);
}
bool host_turns(const OsmosRopeScaling* s, uint32_t rot, double* turns, float* scale) { return rows::turns_of(s, rot, turns, scale); }
bool host_sample(const OsmosSample* a) { return rows::sample_ok(a); }
bool host_launches(uint64_t blocks, uint32_t threads) { return rows::launches(blocks, threads); }
}
