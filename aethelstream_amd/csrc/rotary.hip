// rotary.hip - norms of queries and keys for each head and their rotation by
// position, in one pass, forward and backward, for gfx950 (MI355X).
//
// Rows are the heads of every token of q and k, d elements each (the q/k/v
// products at doublepass/src/forward.rs:174-176 write them; the reference has no
// positions and no norms there):
//   n = w x / rms(x),  rms(x) = sqrt(mean(x^2) + eps)     (n = x without w)
//   pair i < rot / 2 of n turns by t = position f_i:
//     a' = s (a cos t - b sin t),  b' = s (b cos t + a sin t)
// with pairs (i, i + rot / 2), or (2 i, 2 i + 1) if interleaved; elements from rot
// on are not turned.  Backward, from the gradient dy of the result:
//   dn = dy with its pairs turned by -t and scaled by s,  e = w dn,
//   dx = (e - x^ mean(e x^)) / rms,  dw = sum over rows of dn x^,  x^ = x / rms
// (dx = dn without w).  rms is taken again from x, which the pass reads anyway.
//
// Angles.  f_i comes as turns a position in units of 2^-64, so position * f_i
// modulo 2^64 is the fraction of a turn, exact for every 64-bit position; its
// upper 32 bits, signed, are the argument of sine and cosine: at most 2^-25 of a
// turn off.  They are computed once for each token and pair of a workgroup's rows
// and shared through LDS.
//
// A lane holds kNP pairs of a row, both halves of the head, so a rotation needs no
// exchange; 1 to 64 lanes hold a row and sum its squares with DPP adds.  Both
// directions are bound by memory: 4 bytes an element forward in bf16, 6 backward
// with norms.  What is read and written once leaves the caches to others (non-temporal
// accesses: 68 -> 62 us forward of 8192 x 72 heads of 128 in bf16, 4.9 TB/s; backward
// 126 -> 115, with the next tile's loads ahead and fewer elements a lane 102, 4.4 TB/s;
// it waits for memory 64 % of its waves' time, and issues vector instructions 19 %).
#include "row_common.hpp"

namespace nf4s {

constexpr int kRotaryThreads = 256;
constexpr int64_t kMaxHeadSize = 1024;
constexpr int64_t kMaxHeads = 4096;
// Rows of a lane in flight.  The norms' backward holds two tensors and its sums: with
// two rows of 4 + 4 elements a lane four workgroups fit a CU, which together are its
// whole grid.  8192 x 72 heads of 128: 102 us, 108 to 112 with rows of 8 + 8, 133 with
// five workgroups a CU, of which one waits.
constexpr int kRotaryRows = 4, kRotaryBwdRows = 2, kRotaryBwdWgs = 4;
// LDS for the angles of a workgroup's tokens that costs no occupancy.
constexpr int64_t kRotaryAngleBytes = 20 << 10;

// q or k.
struct RotarySide {
  const void *x;   // forward: in; backward: what was normed
  const void *dy;  // backward: in
  void *out;
  int64_t x_token, x_head, dy_token, dy_head, out_token, out_head;  // strides, elements
  const float *w;
  float *part;     // backward: [workgroups of this side][d] sums for dw
  int64_t rows;    // m * heads
  int32_t heads;
  uint32_t magic;  // 2^31 / heads + 1
  int32_t wgs;     // workgroups that share the rows
};

struct RotaryArgs {
  RotarySide side[2];
  const int64_t *positions, *turns;
  int32_t d, rot;
  int32_t lanes_shift;  // log2 of the lanes of a row
  int32_t iters;        // rows of a lane in a tile, up to kRotaryRows
  int32_t angles;       // of a tile's tokens, at most
  float scale, scale_sin, eps;  // scale_sin: negative where the rotation is taken back
};

// Sum over the 2^shift lanes of a row, in each of them.
__device__ __forceinline__ float lanes_sum(float v, int shift) {
  if (shift > 0) v = dpp_add<0xb1>(v);   // quad_perm: lane ^ 1
  if (shift > 1) v = dpp_add<0x4e>(v);   // lane ^ 2
  if (shift > 2) v = dpp_add<0x141>(v);  // half rows mirrored: the other four
  if (shift > 3) v = dpp_add<0x140>(v);  // rows mirrored: the other eight
  if (shift > 4) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    v = __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
  }
  if (shift > 5) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    v = __builtin_bit_cast(float, (uint32_t)s[0]) + __builtin_bit_cast(float, (uint32_t)s[1]);
  }
  return v;
}

__device__ __forceinline__ float rotary_value(uint16_t v) { return bf16_low(v); }
__device__ __forceinline__ float rotary_value(float v) { return v; }
__device__ __forceinline__ void rotary_put(uint16_t *p, float v) {
  *p = (uint16_t)pack_bf16x2(v, 0.0f);
}
__device__ __forceinline__ void rotary_put(float *p, float v) { *p = v; }

// Places of a lane's pairs in a row and the moves between memory and registers.
// kVec: pairs kNP l to kNP l + kNP - 1 of lane l, by vector loads; of pairs that are
// not adjacent all are turned, or none.  Otherwise pairs l + 64 j, element by element.
template <typename T, int kNP, bool kVec, bool kAdj>
struct RotaryLane {
  static constexpr int kWords = kVec ? 2 * kNP * (int)sizeof(T) / 4 : 2 * kNP;
  struct Raw {
    uint32_t v[kWords];
  };
  int first;        // of the lane's pairs
  int pairs, half;  // of a row, of those that turn

  __device__ __forceinline__ int pair(int j) const { return kVec ? first + j : first + 64 * j; }
  __device__ __forceinline__ bool has(int j) const { return pair(kVec ? 0 : j) < pairs; }
  // (Of adjacent pairs a lane may have some that turn.)
  __device__ __forceinline__ bool turns(int j) const {
    return pair(kVec && !kAdj ? 0 : j) < half;
  }
  // Element of pair j's first value, and the distance of its second one.
  __device__ __forceinline__ int place(int j) const {
    const int p = pair(j);
    return kAdj ? 2 * p : p + (p < half ? 0 : half);
  }
  __device__ __forceinline__ int apart(int j) const {
    return kAdj ? 1 : turns(j) ? half : pairs - half;
  }

  __device__ __forceinline__ Raw load(const T *row) const {
    Raw r;
    if constexpr (kVec) {
      constexpr int kHalf = kWords / 2;
      const uint32_t *a = reinterpret_cast<const uint32_t *>(row + place(0));
      const uint32_t *b = kAdj ? a + kHalf
                               : reinterpret_cast<const uint32_t *>(row + place(0) + apart(0));
      if (has(0)) {
        if constexpr (kHalf % 4 == 0) {
#pragma unroll
          for (int i = 0; i < kHalf; i += 4) {
            *reinterpret_cast<u32x4 *>(r.v + i) =
                __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(a + i));
            *reinterpret_cast<u32x4 *>(r.v + kHalf + i) =
                __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(b + i));
          }
        } else if constexpr (kHalf == 1) {
          r.v[0] = __builtin_nontemporal_load(a);
          r.v[1] = __builtin_nontemporal_load(b);
        } else {
          static_assert(kHalf == 2, "two fp32 or four bf16 values");
          *reinterpret_cast<u32x2 *>(r.v) =
              __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(a));
          *reinterpret_cast<u32x2 *>(r.v + 2) =
              __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(b));
        }
      } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) r.v[i] = 0;
      }
    } else {
#pragma unroll
      for (int j = 0; j < kNP; ++j) {
        r.v[2 * j] = r.v[2 * j + 1] = 0;
        if (has(j)) {
          r.v[2 * j] = __builtin_bit_cast(uint32_t, rotary_value(row[place(j)]));
          r.v[2 * j + 1] = __builtin_bit_cast(uint32_t, rotary_value(row[place(j) + apart(j)]));
        }
      }
    }
    return r;
  }

  static __device__ __forceinline__ void values(const Raw &r, float (&a)[kNP], float (&b)[kNP]) {
#pragma unroll
    for (int j = 0; j < kNP; ++j) {
      if constexpr (!kVec || (kAdj && sizeof(T) == 4)) {
        a[j] = __builtin_bit_cast(float, r.v[2 * j]);
        b[j] = __builtin_bit_cast(float, r.v[2 * j + 1]);
      } else if constexpr (kAdj) {
        a[j] = bf16_low(r.v[j]);
        b[j] = bf16_high(r.v[j]);
      } else if constexpr (sizeof(T) == 4) {
        a[j] = __builtin_bit_cast(float, r.v[j]);
        b[j] = __builtin_bit_cast(float, r.v[kNP + j]);
      } else {
        const uint32_t x = r.v[j / 2], y = r.v[kNP / 2 + j / 2];
        a[j] = j % 2 ? bf16_high(x) : bf16_low(x);
        b[j] = j % 2 ? bf16_high(y) : bf16_low(y);
      }
    }
  }

  __device__ __forceinline__ void store(T *row, const float (&a)[kNP],
                                        const float (&b)[kNP]) const {
    if constexpr (kVec) {
      if (!has(0)) return;
      Raw r;
#pragma unroll
      for (int j = 0; j < kNP; ++j) {
        if constexpr (kAdj && sizeof(T) == 4) {
          r.v[2 * j] = __builtin_bit_cast(uint32_t, a[j]);
          r.v[2 * j + 1] = __builtin_bit_cast(uint32_t, b[j]);
        } else if constexpr (kAdj) {
          r.v[j] = pack_bf16x2(a[j], b[j]);
        } else if constexpr (sizeof(T) == 4) {
          r.v[j] = __builtin_bit_cast(uint32_t, a[j]);
          r.v[kNP + j] = __builtin_bit_cast(uint32_t, b[j]);
        } else if (j % 2 == 0) {
          r.v[j / 2] = pack_bf16x2(a[j], a[j + 1]);
          r.v[kNP / 2 + j / 2] = pack_bf16x2(b[j], b[j + 1]);
        }
      }
      constexpr int kHalf = kWords / 2;
      uint32_t *p = reinterpret_cast<uint32_t *>(row + place(0));
      uint32_t *q = kAdj ? p + kHalf : reinterpret_cast<uint32_t *>(row + place(0) + apart(0));
      if constexpr (kHalf % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kHalf; i += 4) {
          __builtin_nontemporal_store(*reinterpret_cast<const u32x4 *>(r.v + i),
                                      reinterpret_cast<u32x4 *>(p + i));
          __builtin_nontemporal_store(*reinterpret_cast<const u32x4 *>(r.v + kHalf + i),
                                      reinterpret_cast<u32x4 *>(q + i));
        }
      } else if constexpr (kHalf == 1) {
        __builtin_nontemporal_store(r.v[0], p);
        __builtin_nontemporal_store(r.v[1], q);
      } else {
        __builtin_nontemporal_store(*reinterpret_cast<const u32x2 *>(r.v),
                                    reinterpret_cast<u32x2 *>(p));
        __builtin_nontemporal_store(*reinterpret_cast<const u32x2 *>(r.v + 2),
                                    reinterpret_cast<u32x2 *>(q));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kNP; ++j)
        if (has(j)) {
          rotary_put(row + place(j), a[j]);
          rotary_put(row + place(j) + apart(j), b[j]);
        }
    }
  }
};

// The rotation alone (its backward is the one by -t), or with the norm forward or
// backward.
enum { kTurn, kNormTurn, kNormTurnBwd };

template <typename T, int kNP, bool kVec, bool kAdj, int kMode>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const RotaryArgs a) {
  using Lane = RotaryLane<T, kNP, kVec, kAdj>;
  using Raw = typename Lane::Raw;
  constexpr bool kNorm = kMode != kTurn, kBwd = kMode == kNormTurnBwd;
  constexpr int kRows = kBwd ? kRotaryBwdRows : kRotaryRows;
  extern __shared__ __attribute__((aligned(16))) f32x2 angles[];  // cos, sin; then dw's sums
  const bool is_k = (int)blockIdx.x >= a.side[0].wgs;
  const RotarySide s = is_k ? a.side[1] : a.side[0];
  const int wg = is_k ? (int)blockIdx.x - a.side[0].wgs : (int)blockIdx.x;
  const int lanes = 1 << a.lanes_shift;
  const int group = (int)threadIdx.x >> a.lanes_shift, groups = kRotaryThreads >> a.lanes_shift;
  const int half = a.rot / 2;
  Lane lane;
  lane.first = ((int)threadIdx.x & (lanes - 1)) * (kVec ? kNP : 1);
  lane.pairs = a.d / 2;
  lane.half = half;

  float wa[kNP], wb[kNP], sa[kNP], sb[kNP];
  if constexpr (kNorm) {
#pragma unroll
    for (int j = 0; j < kNP; ++j) {
      sa[j] = sb[j] = wa[j] = wb[j] = 0.0f;
      if (lane.has(j)) {
        wa[j] = s.w[lane.place(j)];
        wb[j] = s.w[lane.place(j) + lane.apart(j)];
      }
    }
  }
  const float inv_d = 1.0f / (float)a.d;
  const int tile_rows = groups * a.iters;
  const int64_t stride = (int64_t)s.wgs * tile_rows;

  // Rows of a tile, `group` and every `groups`-th behind it.
  struct Tile {
    Raw x[kRows], dy[kBwd ? kRows : 1];
  };
  struct Place {
    int64_t token;  // of the tile's first row
    uint32_t head;
    int rows;
  };
  auto place = [&](int64_t row0) {
    Place p;
    p.token = row0 / s.heads;
    p.head = (uint32_t)(row0 - p.token * s.heads);
    p.rows = s.rows - row0 < tile_rows ? (int)(s.rows - row0) : tile_rows;
    return p;
  };
  // Token (from the tile's first) and head of its row r.
  auto find = [&](const Place &p, int r, int &head) {
    const uint32_t local = p.head + (uint32_t)r;
    const uint32_t t = (uint32_t)(((uint64_t)local * s.magic) >> 31);
    head = (int)(local - t * (uint32_t)s.heads);
    return (int)t;
  };
  auto load = [&](Tile &v, const Place &p) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = group + i * groups;
      if (i >= a.iters || r >= p.rows) continue;
      int head;
      const int64_t token = p.token + find(p, r, head);
      v.x[i] = lane.load(static_cast<const T *>(s.x) + token * s.x_token + head * s.x_head);
      if constexpr (kBwd)
        v.dy[i] = lane.load(static_cast<const T *>(s.dy) + token * s.dy_token + head * s.dy_head);
    }
  };
  // The angles of its tokens.
  auto turn = [&](const Place &p, f32x2 *to) {
    int head;
    const int tokens = find(p, p.rows - 1, head) + 1;
    for (int i = (int)threadIdx.x; i < tokens * half; i += kRotaryThreads) {
      const int t = i / half, c = i - t * half;
      const uint64_t at = (uint64_t)a.positions[p.token + t] * (uint64_t)a.turns[c];
      float sn, cs;
      sincospif((float)(int32_t)(at >> 32) * 0x1p-31f, &sn, &cs);
      to[i] = (f32x2){cs * a.scale, sn * a.scale_sin};
    }
  };
  auto work = [&](const Tile &v, const Place &p, const f32x2 *angles) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int r = group + i * groups;
      if (i >= a.iters || r >= p.rows) continue;
      int head;
      const int t = find(p, r, head);
      float va[kNP], vb[kNP], ya[kNP], yb[kNP];
      const f32x2 *turned = angles + t * half;
      if constexpr (kBwd)
        Lane::values(v.dy[i], va, vb);
      else
        Lane::values(v.x[i], va, vb);
      if constexpr (kMode == kNormTurn) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kNP; ++j)
          sum = __builtin_fmaf(va[j], va[j], __builtin_fmaf(vb[j], vb[j], sum));
        const float inv = 1.0f / __builtin_sqrtf(lanes_sum(sum, a.lanes_shift) * inv_d + a.eps);
#pragma unroll
        for (int j = 0; j < kNP; ++j) {
          va[j] *= inv * wa[j];
          vb[j] *= inv * wb[j];
        }
      }
#pragma unroll
      for (int j = 0; j < kNP; ++j) {
        ya[j] = va[j];
        yb[j] = vb[j];
        if (lane.turns(j)) {
          const f32x2 c = turned[lane.pair(j)];
          ya[j] = __builtin_fmaf(va[j], c.x, -(vb[j] * c.y));
          yb[j] = __builtin_fmaf(vb[j], c.x, va[j] * c.y);
        }
      }
      if constexpr (kBwd) {
        Lane::values(v.x[i], va, vb);
        float sum = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < kNP; ++j) {
          sum = __builtin_fmaf(va[j], va[j], __builtin_fmaf(vb[j], vb[j], sum));
          dot = __builtin_fmaf(ya[j] * wa[j], va[j], __builtin_fmaf(yb[j] * wb[j], vb[j], dot));
        }
        const float inv = 1.0f / __builtin_sqrtf(lanes_sum(sum, a.lanes_shift) * inv_d + a.eps);
        // dx = (e - x (e x) / (d rms^2)) / rms
        const float back = lanes_sum(dot, a.lanes_shift) * inv * inv * inv_d;
#pragma unroll
        for (int j = 0; j < kNP; ++j) {
          const float na = ya[j] * inv, nb = yb[j] * inv;
          sa[j] = __builtin_fmaf(na, va[j], sa[j]);
          sb[j] = __builtin_fmaf(nb, vb[j], sb[j]);
          ya[j] = __builtin_fmaf(va[j], -back * inv, na * wa[j]);
          yb[j] = __builtin_fmaf(vb[j], -back * inv, nb * wb[j]);
        }
      }
      lane.store(static_cast<T *>(s.out) + (p.token + t) * s.out_token + head * s.out_head, ya, yb);
    }
  };

  // The next tile's rows and angles are on their way while one is worked on.
  f32x2 *second = angles + a.angles;
  int64_t row = (int64_t)wg * tile_rows;
  Tile v0, v1;
  Place p0, p1;
  if (row < s.rows) {
    p0 = place(row);
    load(v0, p0);
    turn(p0, angles);
  }
  __syncthreads();
#pragma unroll 1
  for (; row < s.rows; row += 2 * stride) {
    if (row + stride < s.rows) {
      p1 = place(row + stride);
      load(v1, p1);
      turn(p1, second);
    }
    work(v0, p0, angles);
    __syncthreads();
    if (row + stride >= s.rows) break;
    if (row + 2 * stride < s.rows) {
      p0 = place(row + 2 * stride);
      load(v0, p0);
      turn(p0, angles);
    }
    work(v1, p1, second);
    __syncthreads();
  }

  if constexpr (kBwd) {
    // The groups of a wave, then the waves, in a fixed order.
    float *sums = reinterpret_cast<float *>(angles);  // [4][d]
    __syncthreads();
    const int wave = (int)threadIdx.x >> 6;
#pragma unroll
    for (int j = 0; j < kNP; ++j) {
      for (int off = lanes; off < 64; off <<= 1) {
        sa[j] += __shfl_xor(sa[j], off, 64);
        sb[j] += __shfl_xor(sb[j], off, 64);
      }
      if (((int)threadIdx.x & 63) < lanes && lane.has(j)) {
        sums[wave * a.d + lane.place(j)] = sa[j];
        sums[wave * a.d + lane.place(j) + lane.apart(j)] = sb[j];
      }
    }
    __syncthreads();
    for (int i = (int)threadIdx.x; i < a.d; i += kRotaryThreads)
      s.part[(int64_t)wg * a.d + i] =
          sums[i] + sums[a.d + i] + sums[2 * a.d + i] + sums[3 * a.d + i];
  }
}

// dw: the workgroups' sums in order, 16 columns a workgroup, each of its 16 groups
// of threads every 16th.
__global__ void __launch_bounds__(256) rotary_dw_kernel(const float *part_q, const float *part_k,
                                                        int32_t parts_q, int32_t parts_k,
                                                        int32_t d, float *dw_q, float *dw_k) {
  __shared__ float lds[16][17];
  const int col = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int per = (d + 15) / 16;
  const bool is_k = (int)blockIdx.x >= per;
  const int c = ((int)blockIdx.x - (is_k ? per : 0)) * 16 + col;
  const float *part = is_k ? part_k : part_q;
  const int parts = is_k ? parts_k : parts_q;
  float s = 0.0f;
  if (c < d)
#pragma unroll 8
    for (int i = group; i < parts; i += 16) s += part[(int64_t)i * d + c];
  lds[group][col] = s;
  __syncthreads();
  if (group != 0 || c >= d) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += lds[i][col];
  float *dw = is_k ? dw_k : dw_q;
  if (dw != nullptr) dw[c] = s;
}

// How a launch is cut: pairs of a lane, lanes of a row, workgroups of each side.
struct RotaryPlan {
  int np;
  bool vec;
  int lanes_shift, iters;
  int32_t wgs[2];
  int32_t angles;
  int64_t lds;
};

// Workgroups of a launch.  The norms' backward, whose workgroups each write d sums:
// as many as run at once.  The others: one for each tile (8192 x 72 heads of 128: 61
// us; 69 to 82 with fewer that go on to further tiles).
static int64_t rotary_most(bool sums) {
  return sums ? (int64_t)cu_slots() * kRotaryBwdWgs : kMaxThreadsPerLaunch / kRotaryThreads / 2;
}

static RotaryPlan rotary_plan(int64_t m, int64_t d, int64_t rot, const int64_t (&heads)[2],
                              int aligned_pairs, bool adjacent, bool sums) {
  RotaryPlan p{};
  const int64_t pairs = d / 2;
  // Vector accesses of 8, 4 or 2 pairs where rows are whole ones, and of pairs that are
  // not adjacent the halves and what is not turned too.
  int np = sums && aligned_pairs > 4 && pairs <= 256 ? 4 : aligned_pairs;
  while (np > 1 && (d % (2 * np) != 0 || (!adjacent && rot % (2 * np) != 0) || pairs / np > 64))
    np /= 2;
  p.vec = np >= 2;
  int64_t lanes;
  if (p.vec) {
    p.np = np;
    lanes = pairs / np;
  } else {
    p.np = pairs <= 128 ? 2 : 8;
    lanes = pairs < 64 ? pairs : 64;
  }
  while ((1 << p.lanes_shift) < lanes) ++p.lanes_shift;
  const int64_t groups = kRotaryThreads >> p.lanes_shift;
  auto tokens = [&](int64_t h, int64_t iters) {
    const int64_t n = (groups * iters + h - 2) / h + 1;  // a tile may begin inside a token
    return n < m ? n : m;
  };
  const int64_t least = heads[1] > 0 && heads[1] < heads[0] ? heads[1] : heads[0];
  const int64_t rows = m * (heads[0] + heads[1]);
  p.iters = sums ? kRotaryBwdRows : kRotaryRows;
  while (p.iters > 1 && (tokens(least, p.iters) * (rot / 2) * 8 > kRotaryAngleBytes ||
                         rows < groups * p.iters * 2 * cu_slots()))
    p.iters /= 2;
  p.angles = (int32_t)(tokens(least, p.iters) * (rot / 2));
  p.lds = 2 * (int64_t)p.angles * 8;
  if (sums && p.lds < 16 * d) p.lds = 16 * d;
  const int64_t tile = groups * p.iters, most = rotary_most(sums);
  for (int i = 0; i < 2; ++i) {
    const int64_t n = (m * heads[i] + tile - 1) / tile;
    // Shares of the workgroups by rows.
    const int64_t share = heads[i] > 0 ? most * heads[i] / (heads[0] + heads[1]) : 0;
    p.wgs[i] = (int32_t)(n < share ? n : share > 0 ? share : n > 0 ? 1 : 0);
  }
  return p;
}

template <typename T, bool kAdj, int kMode>
static void rotary_launch(const RotaryPlan &p, const RotaryArgs &a, hipStream_t s) {
  auto *kernel = !p.vec ? (p.np == 2 ? rotary_kernel<T, 2, false, kAdj, kMode>
                                     : rotary_kernel<T, 8, false, kAdj, kMode>)
                 : p.np == 8 ? rotary_kernel<T, 8, true, kAdj, kMode>
                 : p.np == 4 ? rotary_kernel<T, 4, true, kAdj, kMode>
                             : rotary_kernel<T, 2, true, kAdj, kMode>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)(p.wgs[0] + p.wgs[1])), dim3(kRotaryThreads),
                     (uint32_t)p.lds, s, a);
}

template <int kMode>
static int32_t rotary_run(const RotaryPlan &p, const RotaryArgs &a, bool bf16, bool adjacent,
                          hipStream_t s) {
  if (bf16)
    adjacent ? rotary_launch<uint16_t, true, kMode>(p, a, s)
             : rotary_launch<uint16_t, false, kMode>(p, a, s);
  else
    adjacent ? rotary_launch<float, true, kMode>(p, a, s)
             : rotary_launch<float, false, kMode>(p, a, s);
  return check_launch("rotary_kernel");
}

static int32_t rotary_shape(int64_t m, int64_t hq, int64_t hk, int64_t d, int64_t rot) {
  if (m < 0 || hq <= 0 || hk < 0 || d <= 0 || rot <= 0)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "bad rotary shape m=%lld heads %lld and %lld of %lld, "
                "%lld turned", (long long)m, (long long)hq, (long long)hk, (long long)d,
                (long long)rot);
  if (d % 2 != 0 || rot % 2 != 0 || rot > d || d > kMaxHeadSize)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE,
                "rotary heads must have an even size up to %lld with an even turned part, got "
                "%lld and %lld", (long long)kMaxHeadSize, (long long)d, (long long)rot);
  if (hq > kMaxHeads || hk > kMaxHeads)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "rotary takes up to %lld heads",
                (long long)kMaxHeads);
  if (m > (int64_t)1 << 32)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "too many rows");
  return NF4S_OK;
}

// Pairs that vector accesses may take at once, by the alignment of a pointer and its
// strides: 8 of them in accesses of 16 bytes, 4 of 16 or 8, 2 of 8 or 4; else 1.
static int aligned_pairs(const void *p, int64_t token, int64_t head, int size, int most) {
  for (; most > 1; most /= 2) {
    const int64_t bytes = most * size < 16 ? most * size : 16;
    if (aligned(p, (uintptr_t)bytes) && token * size % bytes == 0 && head * size % bytes == 0)
      break;
  }
  return most;
}

static RotaryArgs rotary_args(const RotaryPlan &p, int64_t m, int64_t d, int64_t rot,
                              const int64_t (&heads)[2], const float *const (&w)[2],
                              const int64_t *positions, const int64_t *turns, float scale,
                              float scale_sin, float eps) {
  RotaryArgs a{};
  for (int i = 0; i < 2; ++i) {
    RotarySide &s = a.side[i];
    s.w = w[i];
    s.rows = m * heads[i];
    s.heads = heads[i] > 0 ? (int32_t)heads[i] : 1;
    s.magic = (1u << 31) / (uint32_t)s.heads + 1;
    s.wgs = p.wgs[i];
  }
  a.positions = positions;
  a.turns = turns;
  a.d = (int32_t)d;
  a.rot = (int32_t)rot;
  a.lanes_shift = p.lanes_shift;
  a.iters = p.iters;
  a.angles = p.angles;
  a.scale = scale;
  a.scale_sin = scale_sin;
  a.eps = eps;
  return a;
}

}  // namespace nf4s

using namespace nf4s;

extern "C" {

int32_t nf4s_rotary_fwd(const void *q, const void *k, int32_t is_bf16, int64_t m, int64_t hq,
                        int64_t hk, int64_t d, const int64_t *strides, const float *w_q,
                        const float *w_k, float eps, const int64_t *positions,
                        const int64_t *turns, int64_t rot, int32_t interleaved, float scale,
                        void *q_out, void *k_out, void *stream) {
  clear_error();
  const int32_t rc = rotary_shape(m, hq, hk, d, rot);
  if (rc != NF4S_OK || m == 0) return rc;
  if (q == nullptr || q_out == nullptr || strides == nullptr || positions == nullptr ||
      turns == nullptr || (hk > 0 && (k == nullptr || k_out == nullptr)))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
  if (hk > 0 && (w_q != nullptr) != (w_k != nullptr))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "w_q and w_k: both or neither");
  const int size = is_bf16 ? 2 : 4;
  if (!aligned(q, size) || !aligned(k, size) || !aligned(q_out, size) || !aligned(k_out, size) ||
      !aligned(w_q, 4) || !aligned(w_k, 4) || !aligned(positions, 8) || !aligned(turns, 8))
    return fail(NF4S_ERR_MISALIGNED, "rotary: every buffer must be aligned to its elements");
  int np = aligned_pairs(q, strides[0], strides[1], size, 8);
  np = aligned_pairs(q_out, strides[4], strides[5], size, np);
  if (hk > 0) {
    np = aligned_pairs(k, strides[2], strides[3], size, np);
    np = aligned_pairs(k_out, strides[6], strides[7], size, np);
  }
  const int64_t heads[2] = {hq, hk};
  const RotaryPlan p = rotary_plan(m, d, rot, heads, np, interleaved != 0, false);
  const void *in[2] = {q, k};
  void *out[2] = {q_out, k_out};
  const float *w[2] = {w_q, w_k};
  RotaryArgs a = rotary_args(p, m, d, rot, heads, w, positions, turns, scale, scale, eps);
  for (int i = 0; i < 2; ++i) {
    RotarySide &s = a.side[i];
    s.x = in[i];
    s.out = out[i];
    s.x_token = strides[2 * i];
    s.x_head = strides[2 * i + 1];
    s.out_token = strides[4 + 2 * i];
    s.out_head = strides[5 + 2 * i];
  }
  const hipStream_t st = as_stream(stream);
  return w_q != nullptr ? rotary_run<kNormTurn>(p, a, is_bf16 != 0, interleaved != 0, st)
                        : rotary_run<kTurn>(p, a, is_bf16 != 0, interleaved != 0, st);
}

int32_t nf4s_rotary_bwd_workspace_size(int64_t m, int64_t hq, int64_t hk, int64_t d,
                                       int64_t *bytes) {
  clear_error();
  if (bytes == nullptr) return fail(NF4S_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = 0;
  const int32_t rc = rotary_shape(m, hq, hk, d, 2);
  if (rc != NF4S_OK || m == 0) return rc;
  // Whatever the alignment: at most one workgroup for each row.
  const int64_t rows = m * (hq + hk), most = rotary_most(true) + 1;
  *bytes = (rows < most ? rows : most) * d * 4;
  return NF4S_OK;
}

int32_t nf4s_rotary_bwd(const void *dq, const void *dk, const void *q, const void *k,
                        int32_t is_bf16, int64_t m, int64_t hq, int64_t hk, int64_t d,
                        const int64_t *strides, const float *w_q, const float *w_k, float eps,
                        const int64_t *positions, const int64_t *turns, int64_t rot,
                        int32_t interleaved, float scale, void *dq_out, void *dk_out, float *dw_q,
                        float *dw_k, void *workspace, int64_t workspace_bytes, void *stream) {
  clear_error();
  const int32_t rc = rotary_shape(m, hq, hk, d, rot);
  if (rc != NF4S_OK) return rc;
  const bool norm = w_q != nullptr;
  if (hk > 0 && norm != (w_k != nullptr))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "w_q and w_k: both or neither");
  if (norm != (dw_q != nullptr) || (hk > 0 && norm != (dw_k != nullptr)))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "dw_q and dw_k go with w_q and w_k");
  if (!aligned(w_q, 4) || !aligned(w_k, 4) || !aligned(dw_q, 4) || !aligned(dw_k, 4))
    return fail(NF4S_ERR_MISALIGNED, "rotary: every buffer must be aligned to its elements");
  const hipStream_t st = as_stream(stream);
  RotaryPlan p{};
  if (m > 0) {
    if (dq == nullptr || dq_out == nullptr || strides == nullptr || positions == nullptr ||
        turns == nullptr || (hk > 0 && (dk == nullptr || dk_out == nullptr)) ||
        (norm && (q == nullptr || (hk > 0 && k == nullptr))))
      return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
    const int size = is_bf16 ? 2 : 4;
    if (!aligned(dq, size) || !aligned(dk, size) || !aligned(q, size) || !aligned(k, size) ||
        !aligned(dq_out, size) || !aligned(dk_out, size) || !aligned(positions, 8) ||
        !aligned(turns, 8))
      return fail(NF4S_ERR_MISALIGNED, "rotary: every buffer must be aligned to its elements");
    int np = 8;
    const void *ptrs[6] = {dq, dk, norm ? q : nullptr, norm ? k : nullptr, dq_out, dk_out};
    for (int i = 0; i < 6; ++i)
      if (ptrs[i] != nullptr && (hk > 0 || i % 2 == 0))
        np = aligned_pairs(ptrs[i], strides[2 * i], strides[2 * i + 1], size, np);
    const int64_t heads[2] = {hq, hk};
    p = rotary_plan(m, d, rot, heads, np, interleaved != 0, norm);
    const int64_t need = norm ? (int64_t)(p.wgs[0] + p.wgs[1]) * d * 4 : 0;
    if (need > 0 && (workspace == nullptr || workspace_bytes < need))
      return fail(NF4S_ERR_INVALID_ARGUMENT, "rotary backward needs %lld workspace bytes",
                  (long long)need);
    if (need > 0 && !aligned(workspace, 4))
      return fail(NF4S_ERR_MISALIGNED, "workspace must be 4-byte aligned");
    const float *w[2] = {w_q, w_k};
    RotaryArgs a = rotary_args(p, m, d, rot, heads, w, positions, turns, scale, -scale, eps);
    for (int i = 0; i < 2; ++i) {
      RotarySide &s = a.side[i];
      // Without norms the gradient is all that comes in.
      s.x = norm ? ptrs[2 + i] : ptrs[i];
      s.x_token = strides[norm ? 4 + 2 * i : 2 * i];
      s.x_head = strides[norm ? 5 + 2 * i : 2 * i + 1];
      s.dy = ptrs[i];
      s.dy_token = strides[2 * i];
      s.dy_head = strides[2 * i + 1];
      s.out = i == 0 ? dq_out : dk_out;
      s.out_token = strides[8 + 2 * i];
      s.out_head = strides[9 + 2 * i];
      s.part = static_cast<float *>(workspace) + (i == 0 ? 0 : (int64_t)p.wgs[0] * d);
    }
    const int32_t rc2 = norm ? rotary_run<kNormTurnBwd>(p, a, is_bf16 != 0, interleaved != 0, st)
                             : rotary_run<kTurn>(p, a, is_bf16 != 0, interleaved != 0, st);
    if (rc2 != NF4S_OK) return rc2;
  }
  if (!norm) return NF4S_OK;
  // Over no rows the sums are zero.
  const float *part = static_cast<const float *>(workspace);
  const int per = (int)((d + 15) / 16);
  hipLaunchKernelGGL(rotary_dw_kernel, dim3(hk > 0 ? 2 * per : per), dim3(256), 0, st, part,
                     part + (int64_t)p.wgs[0] * d, p.wgs[0], p.wgs[1], (int32_t)d, dw_q, dw_k);
  return check_launch("rotary_dw_kernel");
}

}  // extern "C"
