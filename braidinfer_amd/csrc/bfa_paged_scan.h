// Sums over a wave's lanes for the cut of a ragged batch (bfa_paged.h).
#pragma once

#include "bfa_device.h"
#include "bfa_paged.h"

namespace bfa {

// Inclusive sum over the lanes (row shifts, then the rows' last lanes broadcast), held
// at PAGED_MOST; and what the lanes before hold.
template <int CTRL, int ROWS>
__device__ __forceinline__ int32_t scan_step(int32_t v) {
  return paged_add(v, __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ int32_t scan_lanes(int32_t v) {
  v = scan_step<0x111, 0xF>(v);
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);
  return scan_step<0x143, 0xC>(v);
}
__device__ __forceinline__ int32_t lane_before(int32_t end) {
  const int32_t u = __shfl_up(end, 1);
  return (threadIdx.x & 63) == 0 ? 0 : u;
}

// Sum over the lanes, held likewise; the same in every lane.
__device__ __forceinline__ int32_t sum_lanes(int32_t v) { return __builtin_amdgcn_readlane(scan_lanes(v), 63); }

}  // namespace bfa
