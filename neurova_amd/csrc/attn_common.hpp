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

// Sixteen signed bytes -> two MFMA fragments of eight fp16 (exact): the byte
// with its sign flipped under the exponent of 1024 is 1024 + 128 + c.
__device__ __forceinline__ void codes_to_half(u32x4 w, f16x8& a, f16x8& b) {
  u32x4 lo, hi;
  const f16x2 bias = {(f16)1152.0f, (f16)1152.0f};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = w[i] ^ 0x80808080u;
    const uint32_t x = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
    const uint32_t y = as_u32(as_h2(__builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
    if (i < 2) lo[2 * i] = x, lo[2 * i + 1] = y;
    else hi[2 * i - 4] = x, hi[2 * i - 3] = y;
  }
  a = __builtin_bit_cast(f16x8, lo);
  b = __builtin_bit_cast(f16x8, hi);
}

}  // namespace lb
