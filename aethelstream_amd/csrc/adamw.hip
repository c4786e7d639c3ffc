// adamw.hip - an AdamW step over many tensors in one launch, with the moments in
// 32 or in 8 bits, for gfx950 (MI355X).
//
// The reference's optimizer keeps 8-bit moments with one scale a tensor and steps
// tensor by tensor (galore/kernels/quantize_state.cu:7-59).  For each element, in
// fp32, every operation rounded on its own:
//   g = grad * grad_scale,  m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// p is fp32 or bf16 (rounded to nearest), and an fp32 p may leave a bf16 copy.
//
// 8 bits: blocks of 128 elements of a tensor share one fp32 scale for m and one for
// r = sqrt(v), their largest absolute value (2^-126 at least).  A value y = |x| /
// scale in [0, 1] is held as
//   code = (bits(y + 2^-15) - bits(2^-15)) >> s,  rounded to nearest, ties to even,
// a float with its exponents counted from 2^-15: linear below, a step of 2^-3 (m, s
// = 20, with a sign) or 2^-4 (r, s = 19) of the value above, so a block spans 2^18
// (2^19) with no table and a handful of integer operations.  r of what is not zero
// has at least code 1, as it is divided by in the steps that follow.  The step
// itself uses m and v before they are rounded.  sqrt(v) is correctly rounded, so
// that codes are the format's and not the machine's.
//
// A lane takes 8 elements, so a block is 16 lanes, whose maxima meet in DPP moves.
// All tensors of a launch are one range of chunks; a workgroup finds its tensor by
// bisection in the launch's arguments, which hold their addresses: nothing has to be
// copied to the device before a step.
#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

#include "row_common.hpp"

namespace nf4s {

constexpr int kAdamThreads = 256;
constexpr int kAdamBlock = 128;
constexpr int kAdamEach = 8;   // elements of a lane at once
constexpr int kAdamIter = 2;   // times that in a chunk
constexpr int kAdamChunk = kAdamThreads * kAdamEach * kAdamIter;
constexpr uint32_t kAdamOffset = 0x38000000u;  // 2^-15

enum { kBeta1, kRest1, kBeta2, kRest2, kKeep, kSize, kInvRoot, kEps, kHyper };

struct AdamCommon {
  void *m, *v;  // fp32, or int8 and uint8 codes
  float *m_scale, *v_scale;
  const float *grad_scale;  // device, or NULL
  const float *hyper;       // device, or NULL: `value`
  float value[kHyper];
  int32_t count;
};

// Tensors of a launch: with the common part less than the 4 KB of a kernel's
// arguments.
template <bool kCopy>
struct AdamTable {
  static constexpr int kMost = kCopy ? 98 : 126;
  AdamCommon c;
  void *p[kMost];
  const void *g[kMost];
  uint16_t *copy[kCopy ? kMost : 1];
  uint32_t n[kMost];          // elements
  uint32_t block[kMost];      // first block of its moments
  uint32_t chunk[kMost + 1];  // first chunk, and the last one's end
};
static_assert(sizeof(AdamTable<false>) < 3840 && sizeof(AdamTable<true>) < 3840, "arguments");

__device__ __forceinline__ uint32_t dpp_max16(uint32_t v) {
  auto with = [](uint32_t a, int b) { return a > (uint32_t)b ? a : (uint32_t)b; };
  v = with(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));
  v = with(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
  v = with(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xf, 0xf, true));
  return with(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xf, 0xf, true));
}

// Eight values of either type from p, or those of them below n, one by one.
__device__ __forceinline__ void adam_load(const uint16_t *p, bool whole, uint32_t left,
                                          float (&x)[kAdamEach]) {
  if (whole) {
    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_low(w[i]);
      x[2 * i + 1] = bf16_high(w[i]);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kAdamEach; ++i) x[i] = i < left ? bf16_low(p[i]) : 0.0f;
  }
}
__device__ __forceinline__ void adam_load(const float *p, bool whole, uint32_t left,
                                          float (&x)[kAdamEach]) {
  if (whole) {
    const floatx4 a = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(p));
    const floatx4 b = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(p) + 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kAdamEach; ++i) x[i] = i < left ? p[i] : 0.0f;
  }
}
__device__ __forceinline__ void adam_store(uint16_t *p, bool whole, uint32_t left,
                                           const float (&x)[kAdamEach]) {
  if (whole) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4 *>(p));
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kAdamEach; ++i)
      if (i < left) p[i] = (uint16_t)pack_bf16x2(x[i], 0.0f);
  }
}
__device__ __forceinline__ void adam_store(float *p, bool whole, uint32_t left,
                                           const float (&x)[kAdamEach]) {
  if (whole) {
    __builtin_nontemporal_store((floatx4){x[0], x[1], x[2], x[3]}, reinterpret_cast<floatx4 *>(p));
    __builtin_nontemporal_store((floatx4){x[4], x[5], x[6], x[7]},
                                reinterpret_cast<floatx4 *>(p) + 1);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kAdamEach; ++i)
      if (i < left) p[i] = x[i];
  }
}

// The value of a code's magnitude, over its block's scale.
template <int kShift>
__device__ __forceinline__ float adam_value(uint32_t mag) {
  return __builtin_bit_cast(float, kAdamOffset + (mag << kShift)) -
         __builtin_bit_cast(float, kAdamOffset);
}
template <int kShift>
__device__ __forceinline__ uint32_t adam_code(float y) {
  const uint32_t u =
      __builtin_bit_cast(uint32_t, y + __builtin_bit_cast(float, kAdamOffset)) - kAdamOffset;
  return (u + ((1u << (kShift - 1)) - 1) + ((u >> kShift) & 1)) >> kShift;
}
// A block's scale from its largest absolute value's bits; NaN if that is no number.
__device__ __forceinline__ float adam_scale(uint32_t top) {
  const float t = __builtin_bit_cast(float, top);
  return top >= 0x7f800000u ? __builtin_nanf("") : fmaxf(t, 0x1p-126f);
}

// Moments of the 8 elements from `at`; the moments' buffers are whole blocks long.
__device__ __forceinline__ void adam_moments(const AdamCommon &c, int64_t at, float (&m)[kAdamEach],
                                             float (&v)[kAdamEach], bool bits8) {
  if (bits8) {
    const u32x2 mc = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(c.m) + at);
    const u32x2 vc = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(c.v) + at);
    const float ms = c.m_scale[at / kAdamBlock], vs = c.v_scale[at / kAdamBlock];
#pragma unroll
    for (int i = 0; i < kAdamEach; ++i) {
      const int32_t q = (int32_t)(mc[i / 4] << (24 - 8 * (i % 4))) >> 24;
      const float a = adam_value<20>((uint32_t)(q < 0 ? -q : q)) * ms;
      m[i] = q < 0 ? -a : a;
      const float r = adam_value<19>((vc[i / 4] >> (8 * (i % 4))) & 0xff) * vs;
      v[i] = r * r;
    }
  } else {
    adam_load(static_cast<const float *>(c.m) + at, true, 0, m);
    adam_load(static_cast<const float *>(c.v) + at, true, 0, v);
  }
}

template <typename P, typename G, bool kBits8, bool kCopy>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const AdamTable<kCopy> t) {
  // The tensor whose chunks hold this one.
  int lo = 0, hi = t.c.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.chunk[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const uint32_t n = t.n[lo];
  const uint32_t first = (blockIdx.x - t.chunk[lo]) * kAdamChunk;
  P *p = static_cast<P *>(t.p[lo]);
  const G *g = static_cast<const G *>(t.g[lo]);
  uint16_t *copy = kCopy ? t.copy[lo] : nullptr;
  const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) |
                     reinterpret_cast<uintptr_t>(copy)) & 15) == 0;
  const float *hyper = t.c.hyper;
  float h[kHyper];
#pragma unroll
  for (int i = 0; i < kHyper; ++i) h[i] = hyper != nullptr ? hyper[i] : t.c.value[i];
  const float gs = t.c.grad_scale != nullptr ? *t.c.grad_scale : 1.0f;

  float pv[kAdamIter][kAdamEach], gv[kAdamIter][kAdamEach];
  float m[kAdamIter][kAdamEach], v[kAdamIter][kAdamEach];
#pragma unroll
  for (int k = 0; k < kAdamIter; ++k) {
    const uint32_t e = first + (k * kAdamThreads + threadIdx.x) * kAdamEach;
    const uint32_t left = e < n ? n - e : 0;
    if (left == 0) continue;
    const bool whole = vec && left >= kAdamEach;
    adam_load(p + e, whole, left, pv[k]);
    adam_load(g + e, whole, left, gv[k]);
    adam_moments(t.c, (int64_t)t.block[lo] * kAdamBlock + e, m[k], v[k], kBits8);
  }
#pragma unroll
  for (int k = 0; k < kAdamIter; ++k) {
    const uint32_t e = first + (k * kAdamThreads + threadIdx.x) * kAdamEach;
    const uint32_t left = e < n ? n - e : 0;
    if (!kBits8 && left == 0) continue;
    uint32_t m_top = 0, r_top = 0;
    float r[kAdamEach];
#pragma unroll
    for (uint32_t i = 0; i < kAdamEach; ++i) {
      const float x = gv[k][i] * gs;
      m[k][i] = m[k][i] * h[kBeta1] + x * h[kRest1];
      v[k][i] = v[k][i] * h[kBeta2] + x * x * h[kRest2];
      if (i >= left) m[k][i] = v[k][i] = 0.0f;  // past the tensor's end
      r[i] = __builtin_sqrtf(v[k][i]);
      pv[k][i] = pv[k][i] * h[kKeep] - m[k][i] / (r[i] * h[kInvRoot] + h[kEps]) * h[kSize];
      if (kBits8) {
        const uint32_t a = __builtin_bit_cast(uint32_t, m[k][i]) & 0x7fffffffu;
        const uint32_t b = __builtin_bit_cast(uint32_t, r[i]) & 0x7fffffffu;
        m_top = a > m_top ? a : m_top;
        r_top = b > r_top ? b : r_top;
      }
    }
    const int64_t at = (int64_t)t.block[lo] * kAdamBlock + e;
    if constexpr (kBits8) {
      // All lanes of a block, those past the end with zeros.
      const float ms = adam_scale(dpp_max16(m_top)), rs = adam_scale(dpp_max16(r_top));
      // The last block's lanes past the tensor's end write its codes' rest.
      if (e / kAdamBlock * kAdamBlock >= n) continue;
      const float mi = 1.0f / ms, ri = 1.0f / rs;
      u32x2 mc = {0u, 0u}, vc = {0u, 0u};
#pragma unroll
      for (int i = 0; i < kAdamEach; ++i) {
        const uint32_t a = adam_code<20>(fabsf(m[k][i]) * mi);
        mc[i / 4] |= ((m[k][i] < 0.0f ? 0u - a : a) & 0xff) << (8 * (i % 4));
        uint32_t b = adam_code<19>(r[i] * ri);
        b = r[i] > 0.0f && b == 0 ? 1 : b;
        vc[i / 4] |= (b & 0xff) << (8 * (i % 4));
      }
      *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(t.c.m) + at) = mc;
      *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(t.c.v) + at) = vc;
      if ((threadIdx.x & 15) == 0) {
        t.c.m_scale[at / kAdamBlock] = ms;
        t.c.v_scale[at / kAdamBlock] = rs;
      }
    } else {
      adam_store(static_cast<float *>(t.c.m) + at, true, 0, m[k]);
      adam_store(static_cast<float *>(t.c.v) + at, true, 0, v[k]);
    }
    if (left == 0) continue;
    const bool whole = vec && left >= kAdamEach;
    adam_store(p + e, whole, left, pv[k]);
    if (kCopy) adam_store(copy + e, whole, left, pv[k]);
  }
}

// What 8-bit moments stand for.
__global__ void __launch_bounds__(kAdamThreads) adamw_moments_kernel(AdamCommon c, int64_t blocks,
                                                                     float *m, float *v) {
  const int64_t groups = blocks * (kAdamBlock / kAdamEach);
  for (int64_t i = (int64_t)blockIdx.x * kAdamThreads + threadIdx.x; i < groups;
       i += (int64_t)gridDim.x * kAdamThreads) {
    float a[kAdamEach], b[kAdamEach];
    adam_moments(c, i * kAdamEach, a, b, true);
    adam_store(m + i * kAdamEach, true, 0, a);
    adam_store(v + i * kAdamEach, true, 0, b);
  }
}

// Collects tensors of one kind and launches them.
template <typename P, typename G, bool kBits8, bool kCopy>
struct AdamLaunch {
  using Table = AdamTable<kCopy>;
  Table t;
  hipStream_t stream;

  AdamLaunch(const AdamCommon &c, hipStream_t s) : stream(s) {
    t.c = c;
    t.c.count = 0;
    t.chunk[0] = 0;
  }
  int32_t flush() {
    if (t.c.count == 0) return NF4S_OK;
    hipLaunchKernelGGL((adamw_kernel<P, G, kBits8, kCopy>), dim3(t.chunk[t.c.count]),
                       dim3(kAdamThreads), 0, stream, t);
    t.c.count = 0;
    return check_launch("adamw_kernel");
  }
  // n elements; their moments begin at `block`.
  int32_t add(void *p, const void *g, uint16_t *copy, int64_t n, int64_t block) {
    // Elements of a piece are counted in 32 bits, a launch's threads too.
    constexpr int64_t kPiece = (int64_t)1 << 30;
    for (int64_t at = 0; at < n; at += kPiece) {
      const int64_t k = n - at < kPiece ? n - at : kPiece;
      const uint32_t chunks = (uint32_t)((k + kAdamChunk - 1) / kAdamChunk);
      if (t.c.count == Table::kMost ||
          (int64_t)t.chunk[t.c.count] + chunks > kMaxThreadsPerLaunch / kAdamThreads) {
        const int32_t rc = flush();
        if (rc != NF4S_OK) return rc;
      }
      const int i = t.c.count++;
      t.p[i] = static_cast<P *>(p) + at;
      t.g[i] = static_cast<const G *>(g) + at;
      if (kCopy) t.copy[i] = copy + at;
      t.n[i] = (uint32_t)k;
      t.block[i] = (uint32_t)(block + at / kAdamBlock);
      t.chunk[i + 1] = t.chunk[i] + chunks;
    }
    return NF4S_OK;
  }
};

struct AdamList {
  void *const *params;
  const void *const *grads;
  uint16_t *const *copies;
  const int64_t *sizes;
  const int32_t *types;
  int32_t count;
};

// The tensors of one kind.
template <typename P, typename G, bool kBits8, bool kCopy>
static int32_t adam_kind(const AdamList &l, int32_t type, const AdamCommon &c, hipStream_t s) {
  AdamLaunch<P, G, kBits8, kCopy> launch(c, s);
  int64_t block = 0;
  for (int32_t i = 0; i < l.count; ++i) {
    uint16_t *copy = l.copies != nullptr ? l.copies[i] : nullptr;
    if (l.sizes[i] > 0 && (l.types[i] & 3) == type && (copy != nullptr) == kCopy) {
      const int32_t rc = launch.add(l.params[i], l.grads[i], copy, l.sizes[i], block);
      if (rc != NF4S_OK) return rc;
    }
    block += ceil_div(l.sizes[i], kAdamBlock);
  }
  return launch.flush();
}

template <bool kBits8>
static int32_t adam_run(const AdamList &l, const AdamCommon &c, hipStream_t s) {
  int32_t rc = adam_kind<float, float, kBits8, false>(l, 0, c, s);
  if (rc == NF4S_OK) rc = adam_kind<uint16_t, float, kBits8, false>(l, 1, c, s);
  if (rc == NF4S_OK) rc = adam_kind<float, uint16_t, kBits8, false>(l, 2, c, s);
  if (rc == NF4S_OK) rc = adam_kind<uint16_t, uint16_t, kBits8, false>(l, 3, c, s);
  if (rc != NF4S_OK || l.copies == nullptr) return rc;
  rc = adam_kind<float, float, kBits8, true>(l, 0, c, s);
  if (rc == NF4S_OK) rc = adam_kind<float, uint16_t, kBits8, true>(l, 2, c, s);
  return rc;
}

// Blocks of the moments of all tensors.
static int32_t adam_blocks(const int64_t *sizes, int32_t count, int64_t &blocks) {
  blocks = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (sizes[i] < 0)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "tensor %d has a negative size", (int)i);
    blocks += ceil_div(sizes[i], kAdamBlock);
    if (blocks > (int64_t)0xffffffffu)
      return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "AdamW takes up to 2^32 - 1 blocks of 128 elements");
  }
  return NF4S_OK;
}

// Every tensor's buffers are there and aligned, and no two of what is written
// overlap: each element is updated by one lane, once.
static int32_t adam_buffers(const AdamList &l) {
  std::vector<std::pair<uintptr_t, uintptr_t>> written;
  written.reserve(2 * (size_t)l.count);
  for (int32_t i = 0; i < l.count; ++i) {
    if (l.types[i] < 0 || l.types[i] > 3)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "tensor %d has an unknown type", (int)i);
    if (l.sizes[i] == 0) continue;
    uint16_t *copy = l.copies != nullptr ? l.copies[i] : nullptr;
    if (l.params[i] == nullptr || l.grads[i] == nullptr)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "tensor %d has a NULL buffer", (int)i);
    const int p = l.types[i] & 1 ? 2 : 4, g = l.types[i] & 2 ? 2 : 4;
    if (copy != nullptr && p == 2)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "tensor %d: only an fp32 parameter has a copy",
                  (int)i);
    if (!aligned(l.params[i], p) || !aligned(l.grads[i], g) || !aligned(copy, 2))
      return fail(NF4S_ERR_MISALIGNED, "tensor %d is not aligned to its elements", (int)i);
    const uintptr_t at = reinterpret_cast<uintptr_t>(l.params[i]);
    written.emplace_back(at, at + (uintptr_t)l.sizes[i] * p);
    if (copy != nullptr)
      written.emplace_back(reinterpret_cast<uintptr_t>(copy),
                           reinterpret_cast<uintptr_t>(copy) + (uintptr_t)l.sizes[i] * 2);
  }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].second)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "parameters or copies overlap");
  return NF4S_OK;
}

}  // namespace nf4s

using namespace nf4s;

extern "C" {

int32_t nf4s_adamw_step(void *const *params, const void *const *grads, uint16_t *const *copies,
                        const int64_t *sizes, const int32_t *types, int32_t count, void *m,
                        void *v, float *m_scale, float *v_scale, const float *hyper,
                        const float *device_hyper, const float *grad_scale, void *stream) {
  clear_error();
  if (count < 0) return fail(NF4S_ERR_INVALID_ARGUMENT, "negative count");
  if (count == 0) return NF4S_OK;
  if (params == nullptr || grads == nullptr || sizes == nullptr || types == nullptr ||
      (hyper == nullptr && device_hyper == nullptr))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL list");
  if ((m_scale != nullptr) != (v_scale != nullptr))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "m_scale and v_scale: both or neither");
  int64_t blocks = 0;
  int32_t rc = adam_blocks(sizes, count, blocks);
  if (rc != NF4S_OK || blocks == 0) return rc;
  if (m == nullptr || v == nullptr) return fail(NF4S_ERR_INVALID_ARGUMENT, "m or v is NULL");
  if (!aligned(m, 16) || !aligned(v, 16) || !aligned(m_scale, 4) || !aligned(v_scale, 4) ||
      !aligned(device_hyper, 4) || !aligned(grad_scale, 4))
    return fail(NF4S_ERR_MISALIGNED, "m and v must be 16-byte aligned, scales and scalars 4-byte");
  const AdamList l{params, grads, copies, sizes, types, count};
  try {
    rc = adam_buffers(l);
  } catch (const std::exception &e) {
    rc = fail(NF4S_ERR_INVALID_ARGUMENT, "%d tensors: %s", (int)count, e.what());
  }
  if (rc != NF4S_OK) return rc;
  AdamCommon c{};
  c.m = m;
  c.v = v;
  c.m_scale = m_scale;
  c.v_scale = v_scale;
  c.grad_scale = grad_scale;
  c.hyper = device_hyper;
  for (int i = 0; i < kHyper && device_hyper == nullptr; ++i) c.value[i] = hyper[i];
  const hipStream_t s = as_stream(stream);
  return m_scale != nullptr ? adam_run<true>(l, c, s) : adam_run<false>(l, c, s);
}

int32_t nf4s_adamw_moments(const uint8_t *m, const uint8_t *v, const float *m_scale,
                           const float *v_scale, int64_t blocks, float *m_out, float *v_out,
                           void *stream) {
  clear_error();
  if (blocks < 0) return fail(NF4S_ERR_INVALID_ARGUMENT, "negative block count");
  if (blocks > (int64_t)0xffffffffu)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "AdamW takes up to 2^32 - 1 blocks of 128 elements");
  if (blocks == 0) return NF4S_OK;
  if (m == nullptr || v == nullptr || m_scale == nullptr || v_scale == nullptr ||
      m_out == nullptr || v_out == nullptr)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
  if (!aligned(m, 8) || !aligned(v, 8) || !aligned(m_out, 16) || !aligned(v_out, 16) ||
      !aligned(m_scale, 4) || !aligned(v_scale, 4))
    return fail(NF4S_ERR_MISALIGNED,
                "codes must be 8-byte aligned, moments 16-byte and scales 4-byte");
  AdamCommon c{};
  c.m = const_cast<uint8_t *>(m);
  c.v = const_cast<uint8_t *>(v);
  c.m_scale = const_cast<float *>(m_scale);
  c.v_scale = const_cast<float *>(v_scale);
  const int64_t wgs = ceil_div(blocks * (kAdamBlock / kAdamEach), kAdamThreads);
  const int64_t most = (int64_t)cu_slots() * 32;
  hipLaunchKernelGGL(adamw_moments_kernel, dim3((uint32_t)(wgs < most ? wgs : most)),
                     dim3(kAdamThreads), 0, as_stream(stream), c, blocks, m_out, v_out);
  return check_launch("adamw_moments_kernel");
}

}  // extern "C"
