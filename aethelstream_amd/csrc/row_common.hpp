// row_common.hpp - pieces shared by the row kernels (norms around a block,
// 8-bit checkpoints): chunks of four elements, wave and workgroup sums, the
// checkpoint's decode.
#pragma once

#include "abi_common.hpp"
#include "gemm_common.hpp"
#include "nf4_device.hpp"

namespace nf4s {

// Elements of an 8-bit checkpoint that share a scale, along a row, and the
// chunks of four elements in them.
constexpr int kCkptBlock = 128;
constexpr int kCkptBlockShift = 5;  // log2(kCkptBlock / 4)

// The longest row of the norms and the checkpoint's norm, as of the RMSNorm.
constexpr int64_t kMaxRow = (int64_t)1 << 15;

// A launch's threads are counted in 32 bits.
constexpr int64_t kMaxThreadsPerLaunch = 0xffffffffll;

// Sum over the wave, in every lane and in one fixed order: rotations within
// the rows of 16 lanes, then the two swaps between rows.  About 8 cycles a
// step where a shuffle through LDS takes about 60.
template <int kCtrl>
__device__ __forceinline__ float dpp_add(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, true);
  return v + __builtin_bit_cast(float, o);
}
__device__ __forceinline__ float row_wave_sum(float v) {
  v = dpp_add<0x128>(v);  // row_ror:8
  v = dpp_add<0x124>(v);
  v = dpp_add<0x122>(v);
  v = dpp_add<0x121>(v);
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  v = __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
  const uint32_t c = __builtin_bit_cast(uint32_t, v);
  const auto t = __builtin_amdgcn_permlane32_swap(c, c, false, false);
  return __builtin_bit_cast(float, (uint32_t)t[0]) + __builtin_bit_cast(float, (uint32_t)t[1]);
}

// kN sums over each team of `waves` waves of the workgroup, in every thread of
// the team.  Every wave of the workgroup calls it.  `part` holds kN values for
// each of up to 16 waves; a caller that comes again before every wave has passed
// another barrier takes another one.
template <int kN>
__device__ __forceinline__ void row_team_sum(float (&v)[kN], float *part, int team, int waves) {
#pragma unroll
  for (int i = 0; i < kN; ++i) v[i] = row_wave_sum(v[i]);
  if (waves == 1) return;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < kN; ++i) part[16 * i + (threadIdx.x >> 6)] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    float tot = 0.0f;
    for (int w = 0; w < waves; ++w) tot += part[16 * i + team * waves + w];
    v[i] = tot;
  }
}

// kN sums over the workgroup, in every thread.
template <int kN>
__device__ __forceinline__ void row_block_sum(float (&v)[kN], float *part) {
  row_team_sum(v, part, 0, (int)(blockDim.x >> 6));
}

__device__ __forceinline__ float bf16_low(uint32_t v) {
  return __builtin_bit_cast(float, v << 16);
}
__device__ __forceinline__ float bf16_high(uint32_t v) {
  return __builtin_bit_cast(float, v & 0xffff0000u);
}
__device__ __forceinline__ floatx4 bf16x4_values(u32x2 v) {
  return (floatx4){bf16_low(v.x), bf16_high(v.x), bf16_low(v.y), bf16_high(v.y)};
}
__device__ __forceinline__ u32x2 bf16x4_pack(const floatx4 &v) {
  return (u32x2){pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
}

// Four 8-bit codes times their scale.
__device__ __forceinline__ floatx4 ckpt_values(uint32_t codes, float scale) {
  floatx4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = (float)((int32_t)(codes << (24 - 8 * i)) >> 24) * scale;
  return v;
}

}  // namespace nf4s
