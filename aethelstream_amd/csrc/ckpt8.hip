// ckpt8.hip - activation checkpoints in 8 bits for gfx950 (MI355X).
//
// What the first pass of a double-pass step keeps for the second (the
// reference keeps per-channel int8 activations, doublepass/src/checkpoint.rs
// :21-60 and ramflow/kernels/checkpoint_compress.cu:53-145).  Here a scale
// belongs to 128 elements of one row, so one loud channel costs its own block
// its precision and no other, and a row is coded in one read of it:
//   s = max(absmax * (1 / 127), 2^-126),  q = rint(x * (1 / s)),  x^ = q * s
// in fp32, q in [-127, 127].  The floor of s is the smallest normal number:
// below it 1 / s would overflow, and a block of zeros needs no case of its
// own.  A block that holds an infinity or a NaN has a NaN scale and so reads
// back as NaN throughout: it is not hidden.
//
// All kernels are bound by memory.  Measured at 8192 x 8192: fp32 encode 52 us
// (6.4 TB/s; 60 with one unit a lane, 53 with four), decode 47 (7.1); bf16
// encode 33 (6.1; 45 in units of 4 elements, where the vector instructions of
// maximum, reciprocal and codes set the time), decode 29 (6.9); decode and norm
// 68 (6.9), without writing the residual 36 (5.7).  Past the Infinity Cache (16384
// x 8192) the last writes at 4.6.  Rows that end inside a block take workgroups of
// their own, whose last lanes idle: 8192 rows of 516, 1028 and 2052 columns in fp32
// 7.8, 10.3 and 21.8 us to encode (512, 1024, 2048: 5.8, 8.5 and 15.0).
#include <type_traits>

#include "row_common.hpp"

namespace nf4s {

constexpr int kCkptThreads = 256;
constexpr int kCkptPer = 2;  // units a lane

// The larger of two non-negative values, NaN if either is one: as integers,
// whose order is that of non-negative floats, with NaNs above infinity.
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
  return umax(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xf, 0xf, true));
}
// Largest over the 16 lanes of a row, then of two rows, in every lane of them.
__device__ __forceinline__ uint32_t row16_umax(uint32_t v) {
  v = dpp_umax<0x128>(v);
  v = dpp_umax<0x124>(v);
  v = dpp_umax<0x122>(v);
  return dpp_umax<0x121>(v);
}
__device__ __forceinline__ uint32_t row32_umax(uint32_t v) {
  v = row16_umax(v);
  const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return umax((uint32_t)s[0], (uint32_t)s[1]);
}

// The largest scale of which 127 are finite: one step below the largest fp32
// value / 127, which rounds up.
constexpr float kCkptMaxScale = 0x1.020406p+121f;
constexpr float kOver127 = 1.0f / 127.0f;

// Scale of a block from the bits of its largest magnitude.
__device__ __forceinline__ float ckpt_scale(uint32_t top) {
  if (top >= 0x7f800000u) return __builtin_nanf("");
  return fminf(fmaxf(__builtin_bit_cast(float, top) * kOver127, 0x1p-126f), kCkptMaxScale);
}

// Four codes, q = rint(v * inv): adding 1.5 * 2^23 to the rounded product rounds
// it to an integer (|q| <= 127 in a finite block), whose low byte is the sum's.
// A non-finite block's codes mean nothing, its scale is NaN.
__device__ __forceinline__ uint32_t ckpt_code4(const floatx4 &v, float inv) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float r = fp32_rounded(v[i] * inv) + 12582912.0f;
    b[i] = __builtin_bit_cast(uint32_t, r);
  }
  return perm(perm(b[3], b[2], 0x0c0c0400u), perm(b[1], b[0], 0x0c0c0400u), 0x05040100u);
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// kUnit elements as loaded: 16 bytes of fp32, 8 or 16 of bf16.
template <bool kBf16, int kUnit>
struct CkptUnit {
  static constexpr int kVecs = kUnit / 4;
  typename std::conditional<kBf16, u32x2, floatx4>::type v[kVecs];

  __device__ __forceinline__ void load(const void *x, int64_t at) {
    if constexpr (kUnit == 8) {
      const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(x) + at);
      v[0] = (u32x2){w.x, w.y};
      v[1] = (u32x2){w.z, w.w};
    } else if constexpr (kBf16) {
      v[0] = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(x) + at);
    } else {
      v[0] = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(x) + at);
    }
  }
  // Bits of the largest magnitude, as fp32; a NaN stays above all.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (kBf16) {
      // bf16 magnitudes order as 16-bit integers, two at a time.
      u16x2 t = {0, 0};
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const uint32_t lo = v[i].x & 0x7fff7fffu, hi = v[i].y & 0x7fff7fffu;
        t = __builtin_elementwise_max(t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, lo),
                                                                   __builtin_bit_cast(u16x2, hi)));
      }
      return (uint32_t)(t.x > t.y ? t.x : t.y) << 16;
    } else {
      float t = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = v[0][i];
        t = __builtin_elementwise_maximum(t, __builtin_fabsf(f));
      }
      return __builtin_bit_cast(uint32_t, t) & 0x7fffffffu;
    }
  }
  __device__ __forceinline__ floatx4 values(int i) const {
    if constexpr (kBf16)
      return bf16x4_values(v[i]);
    else
      return v[0];
  }
};

// A lane takes two units (of kUnit elements), 256 apart; a block is 128 / kUnit
// lanes.  Workgroup b takes units [512 (b % segs), ..) of row b / segs; where
// rows are whole blocks the caller passes the tensor as one long row.
template <bool kBf16, int kUnit>
__global__ void __launch_bounds__(kCkptThreads) ckpt_encode_kernel(const void *__restrict__ x,
                                                                  int64_t units, uint32_t segs,
                                                                  int64_t blocks,
                                                                  uint32_t *__restrict__ codes,
                                                                  float *__restrict__ scales) {
  constexpr int kLanes = kCkptBlock / kUnit;
  const int64_t row = blockIdx.x / segs;
  const int64_t c0 = (int64_t)(blockIdx.x % segs) * (kCkptThreads * kCkptPer) + threadIdx.x;
  CkptUnit<kBf16, kUnit> v[kCkptPer];
#pragma unroll
  for (int i = 0; i < kCkptPer; ++i) {
    const int64_t c = c0 + i * kCkptThreads;
    v[i] = {};
    if (c < units) v[i].load(x, row * units + c);
  }
#pragma unroll
  for (int i = 0; i < kCkptPer; ++i) {
    const int64_t c = c0 + i * kCkptThreads;
    const uint32_t top = kLanes == 32 ? row32_umax(v[i].top()) : row16_umax(v[i].top());
    const float s = ckpt_scale(top), inv = 1.0f / s;
    if (c < units) {
      if constexpr (kUnit == 8)
        reinterpret_cast<u32x2 *>(codes)[row * units + c] =
            (u32x2){ckpt_code4(v[i].values(0), inv), ckpt_code4(v[i].values(1), inv)};
      else
        codes[row * units + c] = ckpt_code4(v[i].values(0), inv);
      if (threadIdx.x % kLanes == 0) scales[row * blocks + c / kLanes] = s;
    }
  }
}

template <bool kBf16, int kUnit>
__global__ void __launch_bounds__(kCkptThreads) ckpt_decode_kernel(const uint32_t *codes,
                                                                  const float *scales,
                                                                  int64_t units, uint32_t segs,
                                                                  int64_t blocks, void *y) {
  constexpr int kLanes = kCkptBlock / kUnit;
  const int64_t row = blockIdx.x / segs;
  const int64_t c0 = (int64_t)(blockIdx.x % segs) * (kCkptThreads * kCkptPer) + threadIdx.x;
  u32x2 q[kCkptPer];
  float s[kCkptPer];
#pragma unroll
  for (int i = 0; i < kCkptPer; ++i) {
    const int64_t c = c0 + i * kCkptThreads;
    q[i] = (u32x2){0u, 0u};
    s[i] = 0.0f;
    if (c < units) {
      if constexpr (kUnit == 8)
        q[i] = reinterpret_cast<const u32x2 *>(codes)[row * units + c];
      else
        q[i].x = codes[row * units + c];
      s[i] = scales[row * blocks + c / kLanes];
    }
  }
  auto packed = [](uint32_t codes4, float scale) {
    const floatx4 v = ckpt_values(codes4, scale);
    return bf16x4_pack((floatx4){fp32_rounded(v[0]), fp32_rounded(v[1]), fp32_rounded(v[2]),
                                 fp32_rounded(v[3])});
  };
#pragma unroll
  for (int i = 0; i < kCkptPer; ++i) {
    const int64_t c = c0 + i * kCkptThreads;
    if (c >= units) continue;
    if constexpr (kUnit == 8) {
      const u32x2 a = packed(q[i].x, s[i]), b = packed(q[i].y, s[i]);
      __builtin_nontemporal_store((u32x4){a.x, a.y, b.x, b.y},
                                  reinterpret_cast<u32x4 *>(y) + row * units + c);
    } else if constexpr (kBf16) {
      __builtin_nontemporal_store(packed(q[i].x, s[i]),
                                  reinterpret_cast<u32x2 *>(y) + row * units + c);
    } else {
      __builtin_nontemporal_store(ckpt_values(q[i].x, s[i]),
                                  reinterpret_cast<floatx4 *>(y) + row * units + c);
    }
  }
}

// Decode and RMSNorm of a row in one pass: the recompute's first step, whose
// residual (fp32, if asked for) and GEMM operand (bf16) it writes.  The row
// stays in registers between the sum of squares and the outputs.
template <int kMaxThreads, int kChunks>
__global__ void __launch_bounds__(kMaxThreads) ckpt_norm_kernel(const uint32_t *codes,
                                                                const float *scales,
                                                                const float *w, int32_t chunks,
                                                                int32_t blocks, float eps,
                                                                float *x, uint16_t *y,
                                                                float *rms) {
  __shared__ float part[16];
  const int64_t row = blockIdx.x;
  const int threads = (int)blockDim.x;
  floatx4 v[kChunks];
  float sum[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = (int)threadIdx.x + i * threads;
    v[i] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
    if (c < chunks)
      v[i] = ckpt_values(codes[row * chunks + c], scales[row * blocks + (c >> kCkptBlockShift)]);
  }
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[0] += v[i][j] * v[i][j];
  row_block_sum(sum, part);
  const float r = __builtin_sqrtf(sum[0] / (float)(4 * chunks) + eps);
  const float inv = 1.0f / r;
  if (threadIdx.x == 0) rms[row] = r;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = (int)threadIdx.x + i * threads;
    if (c < chunks) {
      if (x != nullptr)
        __builtin_nontemporal_store(v[i], reinterpret_cast<floatx4 *>(x) + row * chunks + c);
      const floatx4 g = reinterpret_cast<const floatx4 *>(w)[c];
      floatx4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = fp32_rounded(v[i][j] * inv * g[j]);
      __builtin_nontemporal_store(bf16x4_pack(o), reinterpret_cast<u32x2 *>(y) + row * chunks + c);
    }
  }
}

// Checks of a checkpoint's sizes, and the grid of the encode and decode kernels
// in units of `unit` elements.
struct CkptPlan {
  int64_t units, blocks;  // of a row
  uint32_t segs, grid;
};
static int32_t ckpt_plan(int64_t m, int64_t d, int unit, CkptPlan &p) {
  if (m < 0 || d <= 0)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "bad checkpoint shape m=%lld d=%lld", (long long)m,
                (long long)d);
  if (d % 4 != 0)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "checkpoint needs d %% 4 == 0, got %lld",
                (long long)d);
  if (d > ((int64_t)1 << 32) || (m > 0 && d > ((int64_t)1 << 39) / m))
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "checkpoint of %lld x %lld elements is too large",
                (long long)m, (long long)d);
  p.units = d / unit;
  p.blocks = (d + kCkptBlock - 1) / kCkptBlock;
  int64_t rows = m;
  if (d % kCkptBlock == 0) {  // no block ends early: one long row
    p.units *= m;
    p.blocks *= m;
    rows = m > 0 ? 1 : 0;
  }
  const int64_t s = (p.units + kCkptThreads * kCkptPer - 1) / (kCkptThreads * kCkptPer);
  if (rows > 0 && s > kMaxThreadsPerLaunch / kCkptThreads / rows)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "checkpoint of %lld x %lld elements is too large",
                (long long)m, (long long)d);
  p.segs = (uint32_t)s;
  p.grid = (uint32_t)(s * rows);
  return NF4S_OK;
}

// Units of 8 elements for bf16 rows that allow 16-byte accesses (and 8-byte ones
// of the codes), of 4 otherwise.
static int ckpt_unit(const void *x, const void *codes, int64_t d, int32_t is_bf16) {
  return is_bf16 && d % 8 == 0 && aligned(x, 16) && aligned(codes, 8) ? 8 : 4;
}

}  // namespace nf4s

using namespace nf4s;

extern "C" {

int32_t nf4s_ckpt8_encode(const void *x, int32_t x_is_bf16, int64_t m, int64_t d, uint8_t *codes,
                          float *scales, void *stream) {
  clear_error();
  CkptPlan p;
  const int unit = ckpt_unit(x, codes, d, x_is_bf16);
  const int32_t rc = ckpt_plan(m, d, unit, p);
  if (rc != NF4S_OK || m == 0) return rc;
  if (x == nullptr || codes == nullptr || scales == nullptr)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
  if (!aligned(x, x_is_bf16 ? 8 : 16) || !aligned(codes, 4) || !aligned(scales, 4))
    return fail(NF4S_ERR_MISALIGNED,
                "checkpoint: fp32 x must be 16-byte aligned, bf16 x 8-byte, codes and scales "
                "4-byte");
  auto *kernel = unit == 8   ? ckpt_encode_kernel<true, 8>
                 : x_is_bf16 ? ckpt_encode_kernel<true, 4>
                             : ckpt_encode_kernel<false, 4>;
  hipLaunchKernelGGL(kernel, dim3(p.grid), dim3(kCkptThreads), 0, as_stream(stream), x, p.units,
                     p.segs, p.blocks, reinterpret_cast<uint32_t *>(codes), scales);
  return check_launch("ckpt_encode_kernel");
}

int32_t nf4s_ckpt8_decode(const uint8_t *codes, const float *scales, int64_t m, int64_t d, void *x,
                          int32_t x_is_bf16, void *stream) {
  clear_error();
  CkptPlan p;
  const int unit = ckpt_unit(x, codes, d, x_is_bf16);
  const int32_t rc = ckpt_plan(m, d, unit, p);
  if (rc != NF4S_OK || m == 0) return rc;
  if (x == nullptr || codes == nullptr || scales == nullptr)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
  if (!aligned(x, x_is_bf16 ? 8 : 16) || !aligned(codes, 4) || !aligned(scales, 4))
    return fail(NF4S_ERR_MISALIGNED,
                "checkpoint: fp32 x must be 16-byte aligned, bf16 x 8-byte, codes and scales "
                "4-byte");
  auto *kernel = unit == 8   ? ckpt_decode_kernel<true, 8>
                 : x_is_bf16 ? ckpt_decode_kernel<true, 4>
                             : ckpt_decode_kernel<false, 4>;
  hipLaunchKernelGGL(kernel, dim3(p.grid), dim3(kCkptThreads), 0, as_stream(stream),
                     reinterpret_cast<const uint32_t *>(codes), scales, p.units, p.segs, p.blocks,
                     x);
  return check_launch("ckpt_decode_kernel");
}

int32_t nf4s_ckpt8_decode_norm(const uint8_t *codes, const float *scales, const float *w, int64_t m,
                               int64_t d, float eps, float *x, uint16_t *y, float *rms,
                               void *stream) {
  clear_error();
  CkptPlan p;
  const int32_t rc = ckpt_plan(m, d, 4, p);
  if (rc != NF4S_OK) return rc;
  if (d > kMaxRow)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "norm row of %lld elements is too long",
                (long long)d);
  if (m > kMaxThreadsPerLaunch / 1024)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "too many rows");
  if (m == 0) return NF4S_OK;
  if (codes == nullptr || scales == nullptr || w == nullptr || y == nullptr || rms == nullptr)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
  if (!aligned(codes, 4) || !aligned(scales, 4) || !aligned(w, 16) || !aligned(x, 16) ||
      !aligned(y, 8) || !aligned(rms, 4))
    return fail(NF4S_ERR_MISALIGNED,
                "x and w must be 16-byte aligned, y 8-byte, codes, scales and rms 4-byte");
  const int32_t row_chunks = (int32_t)(d / 4);
  const int32_t row_blocks = (int32_t)((d + kCkptBlock - 1) / kCkptBlock);
  // Four chunks a thread up to 1024 threads, then eight.
  const int per = d <= 16384 ? 4 : 8;
  const int threads = ((row_chunks + per - 1) / per + 63) / 64 * 64;
  auto *kernel = per == 8 ? ckpt_norm_kernel<1024, 8>
                          : (threads <= 512 ? ckpt_norm_kernel<512, 4> : ckpt_norm_kernel<1024, 4>);
  hipLaunchKernelGGL(kernel, dim3((uint32_t)m), dim3(threads), 0, as_stream(stream),
                     reinterpret_cast<const uint32_t *>(codes), scales, w, row_chunks, row_blocks,
                     eps, x, y, rms);
  return check_launch("ckpt_norm_kernel");
}

}  // extern "C"
