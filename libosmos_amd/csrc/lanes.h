// libosmos MI355X - sums over a wave's lanes without LDS, for the rows' kernels (include/osmos_rows.h).
#pragma once
#include "common.h"

namespace osm {
namespace rows {

// lanes' values by DPP: row_shr 1, 2, 4, 8, then lane 15 of a row to the next and 31 to the upper half; `none` where there is no
// such lane
template <int STEP>
__device__ inline uint32_t from_below(uint32_t x, uint32_t none) {
  constexpr int ctrl = STEP < 4 ? 0x110 + (1 << STEP) : STEP == 4 ? 0x142 : 0x143;
  constexpr int rows = STEP < 4 ? 0xF : STEP == 4 ? 0xA : 0xC;
  return (uint32_t) __builtin_amdgcn_update_dpp((int) none, (int) x, ctrl, rows, 0xF, false);
}
template <int STEP>
__device__ inline uint64_t from_below(uint64_t x, uint64_t none) {
  return (uint64_t) from_below<STEP>((uint32_t) (x >> 32), (uint32_t) (none >> 32)) << 32 | from_below<STEP>((uint32_t) x, (uint32_t) none);
}
// the sum over the wave, in every lane
template <int STEP = 0>
__device__ inline double wave_total(double x) {
  x += __longlong_as_double((long long) from_below<STEP>((uint64_t) __double_as_longlong(x), (uint64_t) 0));
  if constexpr (STEP < 5) return wave_total<STEP + 1>(x);
  const uint64_t b = (uint64_t) __double_as_longlong(x);
  return __longlong_as_double((long long) ((uint64_t) (uint32_t) __builtin_amdgcn_readlane((int) (b >> 32), 63) << 32 |
                                           (uint32_t) __builtin_amdgcn_readlane((int) b, 63)));
}

}  // namespace rows
}  // namespace osm
