// tr_tile.hpp - LDS tiles whose reduction index is the row (a row-major operand
// whose columns are MFMA operands) and their transposing fragment reads, for
// the gfx950 product dY^T . X.
#pragma once

#include "gemm_common.hpp"
#include "nf4_device.hpp"

namespace nf4s {

// LDS tile: 32 token rows x 256 columns (512 B = 32 units of 16 B per row), or
// 128 columns (16 units) of dy when kMT = 2.  A wave reads one half of the
// columns.  Unit u of row r lives at
// physical unit (u & 16) | ((u & 15) ^ 5 (r % 4)): with it, each 32-lane
// half of a transposed fragment read covers 16 distinct 16-B units of one
// half-row's 64 banks (rows are 512 B or 256 B = 128 or 64 banks apart, so every
// row starts at bank 0), and each 16-lane quarter of a DMA writes one row's 16
// contiguous units.
__device__ __forceinline__ int wg_unit(int row, int u) {
  return (u & 16) | ((u & 15) ^ (5 * (row & 3)));
}

// Byte offset (from its tile's base) of lane `lane`'s first transposed read
// of fragment j: column 32j + lane % 32 of the wave's half h, token rows
// 8 (lane / 32) + 0..3 of sub-step 0.  ds_read_b64_tr_b16 transposes 4 x 4
// blocks of 16-bit values within each 16-lane group: lane i receives element
// i % 4 of the 8 bytes that lane 4e + i / 4 addresses, so lane 4e + c
// addresses row e, columns 4c..4c+3 of the group's 16-column strip.  A second
// read 4 rows lower completes the 8 tokens.
template <int kUnits>
__device__ __forceinline__ uint32_t wg_read_off(int lane, int h, int j) {
  const int l16 = lane & 15, e = l16 >> 2;
  const int row = 8 * (lane >> 5) + e;
  const int u = kUnits / 2 * h + 4 * j + 2 * ((lane >> 4) & 1) + ((l16 >> 1) & 1);
  return (uint32_t)(16 * (kUnits * row + wg_unit(row, u)) + 8 * (l16 & 1));
}

// Fragment (8 tokens of one column, sub-step s) from the tile at `base`, whose
// rows are kUnits 16-byte units long.
template <int kUnits>
__device__ __forceinline__ u32x4 wg_frag(const char *base, uint32_t off, int s) {
  typedef __attribute__((address_space(3))) char lds_char_t;
  typedef __attribute__((address_space(3))) v4i16 lds_v4i16_t;
  lds_char_t *p = (lds_char_t *)const_cast<char *>(base) + off + 256 * kUnits * s;
  const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t *)p);
  const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t *)(p + 64 * kUnits));
  const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
  return (u32x4){l2.x, l2.y, h2.x, h2.y};
}

}  // namespace nf4s
