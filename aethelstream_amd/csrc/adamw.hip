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
// To nearest, a change by less than half the distance of two codes is lost, from 1.6
// to 3.1 % of r and 3.1 to 6.3 % of m, and a step changes r by (1 - b2) / 2 (g^2 / v - 1)
// of it, m by (1 - b1) (g / m - 1).  At 0.95 normal gradients change r by 2.5 % down to
// some 10 % up, enough for the codes' mean to stay within 1 % of fp32 moments; at b2 =
// 0.99 r of a tenth of the gradients stays 2.6 times too large, at 0.999 3.9 times (and
// follows the block's largest value instead), at b1 = 0.99 m does not follow a mean that
// falls to a fifth (2.5 times).  So both are 0.95 at most.
// And m of a zero gradient, whose code would stand for no less than before, takes the
// next lower one.  Its decay by b1 is less than half a code's distance among the lowest
// codes (of up to 2^-16 of the block's largest) and, from 0.945 on, at some of the others:
// held there while sqrt(v) falls too, it would move the parameter for good, by 0.03 lr a
// step on average and up to 0.27 at betas of 0.9 and 0.95 in blocks whose other gradients
// are normal; so it comes to rest, after 2.19 lr on average (32 bits: 2.23).  Only waves
// that have a zero gradient look for it: with a tenth of 512 M gradients zero a step
// takes 1050 to 1072 us where one without takes 965 to 1020.
//
// A lane takes 8 elements, so a block is 16 lanes, whose maxima meet in DPP moves.
// All tensors of a launch are one range of chunks; a workgroup finds its tensor by
// bisection in the launch's arguments, which hold their addresses: nothing has to be
// copied to the device before a step.
//
// Bound by memory: 28 bytes an element in fp32, 30 with a copy (202 M elements: 1068
// us, 5.7 TB/s), 10 with 8-bit moments, bf16 parameters and gradients (512 M elements:
// 931 us, 5.5 TB/s).  The latter was bound by vector instructions, 90 an element (1173
// us), of which the compiler's square root and division were 26; 70 now.  What 8-bit
// moments stand for, 10 bytes an element: 512 M in 955 us (5.4 TB/s; 1308 with 8 values
// a lane, whose 16-byte stores leave every other 16 bytes to the next).
#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

#include "row_common.hpp"

namespace nf4s {

constexpr int kAdamThreads = 256;
constexpr int kAdamBlock = 128;
// Elements of a lane at once: a block's codes are 16 lanes, fp32 rows of 16 bytes.
constexpr int kAdamEach8 = 8, kAdamEach32 = 4;
constexpr int kAdamChunk = 4096;  // elements of a workgroup
constexpr uint32_t kAdamOffset = 0x38000000u;  // 2^-15
constexpr float kAdamMostBeta = 0.95f;  // of 8-bit moments

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

// kN values of either type from p, or `left` of them, one by one.
template <int kN>
__device__ __forceinline__ void adam_load(const uint16_t *p, bool whole, uint32_t left,
                                          float (&x)[kN]) {
  typedef uint32_t words __attribute__((ext_vector_type(kN / 2)));
  if (whole) {
    const words w = __builtin_nontemporal_load(reinterpret_cast<const words *>(p));
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) {
      x[2 * i] = bf16_low(w[i]);
      x[2 * i + 1] = bf16_high(w[i]);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) x[i] = i < left ? bf16_low(p[i]) : 0.0f;
  }
}
template <int kN>
__device__ __forceinline__ void adam_load(const float *p, bool whole, uint32_t left,
                                          float (&x)[kN]) {
  if (whole) {
#pragma unroll
    for (int j = 0; j < kN / 4; ++j) {
      const floatx4 a = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(p) + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * j + i] = a[i];
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) x[i] = i < left ? p[i] : 0.0f;
  }
}
template <int kN>
__device__ __forceinline__ void adam_store(uint16_t *p, bool whole, uint32_t left,
                                           const float (&x)[kN]) {
  typedef uint32_t words __attribute__((ext_vector_type(kN / 2)));
  if (whole) {
    words w;
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    __builtin_nontemporal_store(w, reinterpret_cast<words *>(p));
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i)
      if (i < left) p[i] = (uint16_t)pack_bf16x2(x[i], 0.0f);
  }
}
template <int kN>
__device__ __forceinline__ void adam_store(float *p, bool whole, uint32_t left,
                                           const float (&x)[kN]) {
  if (whole) {
#pragma unroll
    for (int j = 0; j < kN / 4; ++j)
      __builtin_nontemporal_store(
          (floatx4){x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]},
          reinterpret_cast<floatx4 *>(p) + j);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i)
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
  // (The offset's own bits end above the shift: the tie's bit may be taken before it
  // is subtracted.)
  static_assert((kAdamOffset & ((2u << kShift) - 1)) == 0, "offset");
  const uint32_t u = __builtin_bit_cast(uint32_t, y + __builtin_bit_cast(float, kAdamOffset));
  return (u + ((u >> kShift) & 1) + (((1u << (kShift - 1)) - 1) - kAdamOffset)) >> kShift;
}
// A block's scale from its largest absolute value's bits; NaN if that is no number.
__device__ __forceinline__ float adam_scale(uint32_t top) {
  const float t = __builtin_bit_cast(float, top);
  return top >= 0x7f800000u ? __builtin_nanf("") : fmaxf(t, 0x1p-126f);
}
// m of the code in byte i of w, and sqrt(v).
template <int kI>
__device__ __forceinline__ float adam_m(uint32_t w, float scale) {
  const int32_t q = (int32_t)(w << (24 - 8 * kI)) >> 24;
  const int32_t n = -q;
  const float a = adam_value<20>((uint32_t)(q > n ? q : n)) * scale;
  // The sign of q.
  return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, a) & 0x7fffffffu) |
                                       ((uint32_t)q & 0x80000000u));
}
template <int kI>
__device__ __forceinline__ float adam_r(uint32_t w, float scale) {
  return adam_value<19>((w >> (8 * kI)) & 0xff) * scale;
}
// Four codes' low bytes as one word.
__device__ __forceinline__ uint32_t adam_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return perm(perm(d, c, 0x0c0c0400u), perm(b, a, 0x0c0c0400u), 0x05040100u);
}

// The correctly rounded square root of 0 or of a number in [2^-100, 2^120], in six
// instructions instead of sixteen: v y with y = rsqrt(v), and half y times what its
// square leaves.  (Every fp32 number of that range was compared with the correctly
// rounded root; test_adamw_roots_gpu.py compares all of [1, 4) and samples of any size.)
__device__ __forceinline__ float adam_root(float v) {
  const float y = __builtin_amdgcn_rsqf(fmaxf(v, 0x1p-100f));
  const float s = v * y;
  return __builtin_fmaf(__builtin_fmaf(-s, s, v), 0.5f * y, s);
}

template <typename P, typename G, bool kBits8, bool kCopy>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const AdamTable<kCopy> t) {
  constexpr int kEach = kBits8 ? kAdamEach8 : kAdamEach32;
  constexpr int kIter = kAdamChunk / kAdamThreads / kEach;
  // The tensor whose chunks hold this one.
  int lo = 0, hi = t.c.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.chunk[mid] <= blockIdx.x) lo = mid;
    else hi = mid;
  }
  const uint32_t n = t.n[lo];
  const uint32_t first = (blockIdx.x - t.chunk[lo]) * kAdamChunk;
  const int64_t base = (int64_t)t.block[lo] * kAdamBlock;  // of the tensor's moments
  P *p = static_cast<P *>(t.p[lo]);
  const G *g = static_cast<const G *>(t.g[lo]);
  uint16_t *copy = kCopy ? t.copy[lo] : nullptr;
  const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) |
                     reinterpret_cast<uintptr_t>(copy)) & 15) == 0;
  const float *hyper = t.c.hyper;
  float h[kHyper];
#pragma unroll
  for (int i = 0; i < kHyper; ++i) h[i] = hyper != nullptr ? hyper[i] : t.c.value[i];
  float gs = t.c.grad_scale != nullptr ? *t.c.grad_scale : 1.0f;
  // Coefficients of the device that 8-bit moments do not take: all is NaN.
  if (kBits8 && !(h[kBeta1] <= kAdamMostBeta && h[kBeta2] <= kAdamMostBeta))
    gs = __builtin_nanf("");

  // All loads, then all else.
  float pv[kIter][kEach], gv[kIter][kEach], mv[kIter][kEach], vv[kIter][kEach];
  u32x2 mc[kIter], vc[kIter];
  float ms[kIter], vs[kIter];
#pragma unroll
  for (int k = 0; k < kIter; ++k) {
    const uint32_t e = first + (k * kAdamThreads + threadIdx.x) * kEach;
    const uint32_t left = e < n ? n - e : 0;
    if (left == 0) continue;
    const bool whole = vec && left >= kEach;
    adam_load(p + e, whole, left, pv[k]);
    adam_load(g + e, whole, left, gv[k]);
    const int64_t at = base + e;
    if constexpr (kBits8) {
      mc[k] = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(t.c.m) + at);
      vc[k] = *reinterpret_cast<const u32x2 *>(static_cast<const uint8_t *>(t.c.v) + at);
      ms[k] = t.c.m_scale[at / kAdamBlock];
      vs[k] = t.c.v_scale[at / kAdamBlock];
    } else {
      adam_load(static_cast<const float *>(t.c.m) + at, true, 0, mv[k]);
      adam_load(static_cast<const float *>(t.c.v) + at, true, 0, vv[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < kIter; ++k) {
    const uint32_t e = first + (k * kAdamThreads + threadIdx.x) * kEach;
    const uint32_t left = e < n ? n - e : 0;
    if (!kBits8 && left == 0) continue;
    float (&m)[kEach] = mv[k], (&v)[kEach] = vv[k], (&x)[kEach] = pv[k];
    float smallest = __builtin_inff();  // |gradient|
    if constexpr (kBits8) {
      static_for<0, kEach>([&](auto I) {
        constexpr int i = decltype(I)::value;
        m[i] = adam_m<i % 4>(mc[k][i / 4], ms[k]);
        const float q = adam_r<i % 4>(vc[k][i / 4], vs[k]);
        v[i] = q * q;
      });
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const float d = gv[k][i] * gs;
      if (kBits8) smallest = fminf(smallest, fabsf(d));
      m[i] = m[i] * h[kBeta1] + d * h[kRest1];
      v[i] = v[i] * h[kBeta2] + d * d * h[kRest2];
    }
    if (left < kEach) {  // zeros past the tensor's end
#pragma unroll
      for (uint32_t i = 0; i < kEach; ++i)
        if (i >= left) m[i] = v[i] = 0.0f;
    }
    float r[kEach];
    uint32_t m_top = 0, r_top = 0, v_least = ~0u;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      r[i] = adam_root(v[i]);
      // Zero as the largest.
      const uint32_t b = __builtin_bit_cast(uint32_t, v[i]) - 1;
      v_least = b < v_least ? b : v_least;
      const uint32_t rb = __builtin_bit_cast(uint32_t, r[i]);
      r_top = rb > r_top ? rb : r_top;
      const uint32_t mb = __builtin_bit_cast(uint32_t, m[i]) & 0x7fffffffu;
      m_top = mb > m_top ? mb : m_top;
    }
    // Outside the quick root's range (2^-100 to 2^120; NaN), for the whole wave.
    if (__ballot(v_least < 0x0d800000u - 1 || r_top >= 0x5d800000u) != 0) {
      r_top = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        r[i] = __builtin_sqrtf(v[i]);
        const uint32_t rb = __builtin_bit_cast(uint32_t, r[i]) & 0x7fffffffu;
        r_top = rb > r_top ? rb : r_top;
      }
    }
    // The quotient by the reciprocal, one step (2^-23) of the update at most.
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      x[i] = x[i] * h[kKeep] -
             m[i] * __builtin_amdgcn_rcpf(r[i] * h[kInvRoot] + h[kEps]) * h[kSize];
    const int64_t at = base + e;
    if constexpr (kBits8) {
      // All lanes of a block, those past the end with zeros.
      const float scale_m = adam_scale(dpp_max16(m_top)), scale_r = adam_scale(dpp_max16(r_top));
      // The last block's lanes past the tensor's end write its codes' rest.
      if (e / kAdamBlock * kAdamBlock >= n) continue;
      const float mi = 1.0f / scale_m, ri = 1.0f / scale_r;
      uint32_t a[kEach], b[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) a[i] = adam_code<20>(fabsf(m[i]) * mi);
      if (__ballot(smallest == 0.0f) != 0) {
        static_for<0, kEach>([&](auto I) {
          constexpr int i = decltype(I)::value;
          const float before = fabsf(adam_m<i % 4>(mc[k][i / 4], ms[k]));
          if (gv[k][i] * gs == 0.0f && a[i] > 0 && adam_value<20>(a[i]) * scale_m >= before)
            --a[i];
        });
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const uint32_t sign = (uint32_t)(__builtin_bit_cast(int32_t, m[i]) >> 31);
        a[i] = (a[i] ^ sign) - sign;
        // At least 1 where r is not zero.
        const uint32_t some = __builtin_bit_cast(uint32_t, r[i]);
        const uint32_t least = some < 1u ? some : 1u, c = adam_code<19>(r[i] * ri);
        b[i] = c > least ? c : least;
      }
      const u32x2 mo = {adam_bytes(a[0], a[1], a[2], a[3]), adam_bytes(a[4], a[5], a[6], a[7])};
      const u32x2 vo = {adam_bytes(b[0], b[1], b[2], b[3]), adam_bytes(b[4], b[5], b[6], b[7])};
      *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(t.c.m) + at) = mo;
      *reinterpret_cast<u32x2 *>(static_cast<uint8_t *>(t.c.v) + at) = vo;
      if ((threadIdx.x & 15) == 0) {
        t.c.m_scale[at / kAdamBlock] = scale_m;
        t.c.v_scale[at / kAdamBlock] = scale_r;
      }
    } else {
      adam_store(static_cast<float *>(t.c.m) + at, true, 0, m);
      adam_store(static_cast<float *>(t.c.v) + at, true, 0, v);
    }
    if (left == 0) continue;
    const bool whole = vec && left >= kEach;
    adam_store(p + e, whole, left, x);
    if (kCopy) adam_store(copy + e, whole, left, x);
  }
}

// What 8-bit moments stand for: a lane four of each at once, four times.
constexpr int kAdamWords = 4;
__global__ void __launch_bounds__(kAdamThreads) adamw_moments_kernel(
    const uint32_t *m, const uint32_t *v, const float *m_scale, const float *v_scale,
    int64_t words, floatx4 *m_out, floatx4 *v_out) {
  for (int64_t first = (int64_t)blockIdx.x * kAdamThreads * kAdamWords + threadIdx.x;
       first < words; first += (int64_t)gridDim.x * kAdamThreads * kAdamWords) {
    uint32_t a[kAdamWords], b[kAdamWords];
    float ms[kAdamWords], vs[kAdamWords];
#pragma unroll
    for (int k = 0; k < kAdamWords; ++k) {
      const int64_t i = first + k * kAdamThreads;
      if (i < words) {
        a[k] = m[i];
        b[k] = v[i];
        ms[k] = m_scale[i / (kAdamBlock / 4)];
        vs[k] = v_scale[i / (kAdamBlock / 4)];
      }
    }
#pragma unroll
    for (int k = 0; k < kAdamWords; ++k) {
      const int64_t i = first + k * kAdamThreads;
      if (i >= words) break;
      floatx4 x, y;
      static_for<0, 4>([&](auto J) {
        constexpr int j = decltype(J)::value;
        x[j] = adam_m<j>(a[k], ms[k]);
        const float r = adam_r<j>(b[k], vs[k]);
        y[j] = r * r;
      });
      __builtin_nontemporal_store(x, m_out + i);
      __builtin_nontemporal_store(y, v_out + i);
    }
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

// Every tensor's buffers are there and aligned, no two of what is written overlap, as
// each element is updated by one lane, once, and no gradient lies in what is written,
// but for one that is its own parameter.
static int32_t adam_buffers(const AdamList &l, const AdamCommon &c, int64_t blocks) {
  typedef std::pair<uintptr_t, uintptr_t> Range;
  std::vector<Range> written;
  written.reserve(2 * (size_t)l.count + 4);
  auto add = [&](const void *p, int64_t bytes) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    if (p != nullptr) written.emplace_back(at, at + (uintptr_t)bytes);
  };
  const bool bits8 = c.m_scale != nullptr;
  add(c.m, blocks * kAdamBlock * (bits8 ? 1 : 4));
  add(c.v, blocks * kAdamBlock * (bits8 ? 1 : 4));
  add(c.m_scale, blocks * 4);
  add(c.v_scale, blocks * 4);
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
    add(l.params[i], l.sizes[i] * p);
    add(copy, l.sizes[i] * 2);
  }
  std::sort(written.begin(), written.end());
  for (size_t i = 1; i < written.size(); ++i)
    if (written[i].first < written[i - 1].second)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "parameters, copies or moments overlap");
  for (int32_t i = 0; i < l.count; ++i) {
    if (l.sizes[i] == 0) continue;
    const int p = l.types[i] & 1 ? 2 : 4, g = l.types[i] & 2 ? 2 : 4;
    if (l.grads[i] == l.params[i] && p == g) continue;
    const uintptr_t from = reinterpret_cast<uintptr_t>(l.grads[i]);
    const uintptr_t to = from + (uintptr_t)l.sizes[i] * g;
    // The first range that ends behind the gradient's begin.
    const auto at = std::upper_bound(
        written.begin(), written.end(), from,
        [](uintptr_t v, const Range &r) { return v < r.second; });
    if (at != written.end() && at->first < to)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "gradient %d lies in what is written", (int)i);
  }
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
  if (m_scale != nullptr && device_hyper == nullptr &&
      !(hyper[kBeta1] <= kAdamMostBeta && hyper[kBeta2] <= kAdamMostBeta))
    return fail(NF4S_ERR_INVALID_ARGUMENT,
                "8-bit moments take beta1 and beta2 up to 0.95, got %g and %g",
                (double)hyper[kBeta1], (double)hyper[kBeta2]);
  const AdamList l{params, grads, copies, sizes, types, count};
  AdamCommon c{};
  c.m = m;
  c.v = v;
  c.m_scale = m_scale;
  c.v_scale = v_scale;
  c.grad_scale = grad_scale;
  c.hyper = device_hyper;
  for (int i = 0; i < kHyper && device_hyper == nullptr; ++i) c.value[i] = hyper[i];
  try {
    rc = adam_buffers(l, c, blocks);
  } catch (const std::exception &e) {
    rc = fail(NF4S_ERR_INVALID_ARGUMENT, "%d tensors: %s", (int)count, e.what());
  }
  if (rc != NF4S_OK) return rc;
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
  const int64_t words = blocks * (kAdamBlock / 4);
  const int64_t wgs = ceil_div(words, kAdamThreads * kAdamWords);
  const int64_t most = (int64_t)cu_slots() * 4096;
  hipLaunchKernelGGL(adamw_moments_kernel, dim3((uint32_t)(wgs < most ? wgs : most)),
                     dim3(kAdamThreads), 0, as_stream(stream),
                     reinterpret_cast<const uint32_t *>(m), reinterpret_cast<const uint32_t *>(v),
                     m_scale, v_scale, words, reinterpret_cast<floatx4 *>(m_out),
                     reinterpret_cast<floatx4 *>(v_out));
  return check_launch("adamw_moments_kernel");
}

}  // extern "C"
