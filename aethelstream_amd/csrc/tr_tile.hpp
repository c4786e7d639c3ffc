// tr_tile.hpp - the transposing fragment read of gfx950's bf16 products whose
// operand lies in LDS with the reduction index as the row.
#pragma once

#include "gemm_common.hpp"
#include "nf4_device.hpp"

namespace nf4s {

// Eight consecutive k of one column from byte `off` of `base`, rows of kUnits
// 16-byte units.  ds_read_b64_tr_b16 transposes 4 x 4 blocks of 16-bit values
// within each 16-lane group: lane i receives element i % 4 of the 8 bytes that
// lane 4e + i / 4 addresses, so lane 4e + c addresses row e, columns 4c..4c+3 of
// the group's 16 columns.  The second read, 4 rows lower, completes the 8.
template <int kUnits>
__device__ __forceinline__ u32x4 tr_frag(const char *base, uint32_t off) {
  typedef __attribute__((address_space(3))) char lds_char_t;
  typedef __attribute__((address_space(3))) v4i16 lds_v4i16_t;
  lds_char_t *p = (lds_char_t *)const_cast<char *>(base) + off;
  const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t *)p);
  const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t *)(p + 64 * kUnits));
  const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
  return (u32x4){l2.x, l2.y, h2.x, h2.y};
}

}  // namespace nf4s
