// Device helpers shared by the attention kernels: the 8-bit cache's writer and
// reader, and the prompt attention.
#pragma once

#include "lb_common.hpp"

namespace lb {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ int lane_id() { return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); }

__device__ __forceinline__ uint32_t from_lane(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(lane << 2, (int)v);
}
__device__ __forceinline__ float from_lane(float v, int lane) {
  return __builtin_bit_cast(float, from_lane(__builtin_bit_cast(uint32_t, v), lane));
}

// Inclusive prefix sum over the wave: four shifted adds inside each row of 16
// lanes, then the rows' last lanes carried on.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}

// One word through a resource with the device-coherence bit (publish16 and
// collect16 move four).
__device__ __forceinline__ float collect4(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, kSc1));
}

}  // namespace lb
