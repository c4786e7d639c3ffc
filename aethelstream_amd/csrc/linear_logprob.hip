// linear_logprob.hip - log probabilities of given tokens under a linear head, the
// entropy of each token's distribution and its most likely alternatives, with the
// gradients of the first two, for gfx950 (MI355X).
//
// x [M, d] and w [V, d] bf16 (the head of doublepass/src/loss.rs and
// doublepass/kernels/fused_ce.cu:71-207, whose cross entropy is linear_ce.hip's):
//   z = x . w^T,  L = log sum_c exp z_c,  logp = z_t - L,  l_c = z_c - L
//   H = -sum_c exp(l_c) l_c
//   top k: the k largest z_c, equal ones by their index, with their l_c
//   G_c = ([c = t] a - exp(l_c) (a + h (l_c + H))) / C,  a = dlogp, h = dH,
//   dx = C G . w,  dw = C G^T . x
// C is the largest |a| (of |h| if that is next to nothing), kept out of the bf16 G as in
// the cross entropy.  Products accumulate in fp32; maxima, sums and results are fp32.
// G is rounded to bf16 because both products are bf16 MFMAs: as two bf16 numbers it would
// take each of them twice, some 6 and 6 ms more of the 19.8 below.  With all else in 64
// bits, that rounding and the result's own (0.0017, relative) leave dx of 77 tokens, 32000
// x 4096, 0.00242 from the exact gradient and dw 0.00177, of 4096 tokens, 128000 x 8192,
// 0.00233 and 0.00228: what the kernels have, to four digits.  (Up to 0.0027 of other
// shapes; a dw in fp32 has G's part alone, 0.0007 and 0.0016 of these.)
//
// Forward: the tiles of the cross entropy, a lane holding one token's columns.  A
// half tile leaves its maximum, its sum of exponentials and the sum of e y with y =
// (z - maximum) log2(e) <= 0, terms of one sign, so that
//   H = log S - ln 2 T / S
// loses nothing to cancellation.
// Alternatives: the k largest logits of a token lie in the k half tiles of largest
// maximum (earlier ones first among equals): any other one has k logits before all
// of its own.  So the logits of the present piece of the vocabulary are stored in
// fp32, but for half tiles whose maximum does not exceed the k-th best of the pieces
// before, and one wave a token picks half tiles by their maxima and reads about k of
// them.  Later columns lose a tie, so what is skipped is never needed.
// Gradients: G by pieces of the vocabulary, from the logits made again or, where the
// forward kept them (the caller's memory), from those: a read of 4 M V bytes for a
// product of 2 M V d.
//
// Measured at 4096 tokens, 128000 x 8192: forward 6.2 ms with the logits kept (2 GB;
// 6.0 without), G of 32000 columns 160 us from them (4.9 TB/s; 1640 made again), dx
// and dw of a piece 1505 and 1540; all of it 19.2 to 19.8 ms, 25.1 with the logits made
// again.  77 tokens, 32000 x 4096: 221 us (258).  1000 tokens, 50021 x 5120 with 20
// alternatives: logits 425 + 30 us (the stores of 200 MB are about 25 of them),
// alternatives 20, sums 7.  One token, 32000 x 4096 with 8: 63 us, of which W takes 50
// (5.2 TB/s).
#include "linear_head.hpp"

namespace nf4s {

constexpr int kLpTop = 32;  // alternatives at most
// Stored logits of a piece: what the Infinity Cache holds between the two kernels.
constexpr int64_t kLpPieceBytes = (int64_t)256 << 20;
// Columns of a piece, whose half tiles' maxima a wave holds in LDS: 16 KB for 64 columns
// each.  Half tiles of 32 are at most four a CU (lp_tiles), 1024 of them: 4 KB alone, 12
// behind whole rounds, whose half tiles have 128.
constexpr int64_t kLpPieceCols = 1 << 18;
constexpr int64_t kLpSelectLds = 64 << 10;

struct LpLogits {
  const uint16_t *x, *w;  // w at the launch's first row
  const int64_t *targets;
  int64_t M, d;
  int64_t v0;   // first column of the launch
  int32_t vn;   // its columns
  int64_t V, ignore;
  int32_t tiles_l, tiles_r;
  // forward
  floatx2 *part;  // [2 tiles_r][M] maximum, sum
  float *ent;     // [2 tiles_r][M] sum of e y
  float *zt;      // [M] logit of the target
  float *z;       // [2 tiles_r][M][32 kNT] logits, or NULL
  const uint64_t *best;  // [M][k] of the pieces before, or NULL
  int32_t k;
  // backward
  const float *lse, *entropy, *dlogp, *dentropy;  // entropy, dentropy: NULL if none
  const float *common;
  uint16_t *g;
  int64_t ldg, gcols;
};

// fp32 values in the order of unsigned integers from 1 on (NaN last); 0: none.
__device__ __forceinline__ uint32_t lp_order(float v) {
  const float u = v + 0.0f;  // -0 as 0
  const uint32_t b = u != u ? 0x7fc00000u : __builtin_bit_cast(uint32_t, u);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t o) {
  return __builtin_bit_cast(float, o ^ (o >> 31 != 0 ? 0x80000000u : 0xffffffffu));
}
// Larger values first, then smaller columns.
__device__ __forceinline__ uint64_t lp_key(uint32_t order, uint32_t column) {
  return order == 0 ? 0 : (uint64_t)order << 32 | (uint32_t)~column;
}
// At least -1e4, where exp2 is 0; NaN stays.
__device__ __forceinline__ float lp_floor(float y) { return y < -1e4f ? -1e4f : y; }

// What a token's gradients of the logits need, divided by C.
struct LpToken {
  float lse, da, dh, base;  // base: dlogp + dentropy * entropy
  bool none;                // both gradients are zero
};
__device__ __forceinline__ LpToken lp_token(const LpLogits &a, int64_t row, bool here, int64_t t) {
  LpToken k;
  k.lse = here ? a.lse[row] : 0.0f;
  const bool given = t != a.ignore;
  k.da = here && given ? a.dlogp[row] / *a.common : 0.0f;
  k.dh = here && a.dentropy != nullptr ? a.dentropy[row] / *a.common : 0.0f;
  k.none = k.da == 0.0f && k.dh == 0.0f;
  if (given && (t < 0 || t >= a.V)) k.da = __builtin_nanf("");
  k.base = k.dh == 0.0f ? k.da : k.da + k.dh * a.entropy[row];
  return k;
}
// G of a logit that is not the given token's.
__device__ __forceinline__ float lp_grad(const LpToken &k, float z) {
  // Past -1e4 the exponential is zero whatever is behind it.
  const float l = lp_floor(z - k.lse);
  return -exp_of(l) * (k.base + k.dh * l);
}

template <int kMT, int kNT, bool kGrad>
__global__ void __launch_bounds__(kGcThreads, kMT == 1 ? 2 : 1) lp_logits_kernel(const LpLogits a) {
  using Core = GcCore<kMT, kNT, false, false>;
  __shared__ __attribute__((aligned(16))) char lds[Core::kLdsBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  int tl, tr;
  gc_tile(blockIdx.x, a.tiles_l, a.tiles_r, kCeStrip, tl, tr);
  const int64_t l0 = (int64_t)tl * Core::kTileL;
  const int r0 = tr * Core::kTileR;
  const int64_t lrows = a.M - l0 < Core::kTileL ? a.M - l0 : Core::kTileL;
  const int rrows = a.vn - r0 < Core::kTileR ? a.vn - r0 : Core::kTileR;
  Core core;
  core.run(gc_along(a.x + l0 * a.d, a.d, lrows, a.d),
           gc_along(a.w + (int64_t)r0 * a.d, a.d, rrows, a.d), a.d, lds, lane, wave);

  // Columns and tokens of a lane: as in ce_logits_kernel.
  const int64_t row0 = l0 + 32 * kMT * (wave >> 1);
  const int c0 = 32 * kNT * (wave & 1);
  const int cols = rrows - c0;
#pragma unroll
  for (int mt = 0; mt < 2 * kMT; ++mt) {
    // One block of 16 tokens at a time: interleaved, the blocks spill.
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(lane));
    floatx4 (&z)[2 * kNT] = core.acc[mt];
    const int grp = lane >> 4;
    if (cols < 32 * kNT) {  // columns past the vocabulary
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * nt + 4 * grp + i >= cols) z[nt][i] = -__builtin_inff();
    }
    const int64_t row = row0 + 16 * mt + (lane & 15);
    const bool here = row < a.M;
    const int64_t t = here ? a.targets[row] : a.ignore;
    // The target's register among this lane's, or -1.
    const int64_t rel = t - (a.v0 + r0 + c0);
    const bool mine = t != a.ignore && rel >= 0 && rel < 32 * kNT && rel < cols &&
                      (((int)rel >> 2) & 3) == grp;
    const int at = mine ? 4 * ((int)rel >> 4) + ((int)rel & 3) : -1;
    if constexpr (!kGrad) {
      if (__ballot(mine) != 0) {
        float zt = 0.0f;
#pragma unroll
        for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) zt = at == 4 * nt + i ? z[nt][i] : zt;
        if (mine) a.zt[row] = zt;
      }
      float top = -__builtin_inff();
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, z[nt][i]);
      top = over_groups(top, [](float x, float y) { return fmaxf(x, y); });
      const int64_t slice = (int64_t)(2 * tr + (wave & 1)) * a.M + row;
      if (a.z != nullptr) {
        const bool keep =
            here && (a.best == nullptr ||
                     lp_order(top) > (uint32_t)(a.best[row * a.k + a.k - 1] >> 32));
        if (__ballot(keep) != 0 && keep) {
          float *out = a.z + slice * (32 * kNT) + 4 * grp;
#pragma unroll
          for (int nt = 0; nt < 2 * kNT; ++nt)
            *reinterpret_cast<floatx4 *>(out + 16 * nt) = z[nt];
        }
      }
      // Nothing but -inf: any finite reference gives a sum of 0.
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f, ent = 0.0f;
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = lp_floor((z[nt][i] - ref) * kLog2e);
          const float e = __builtin_amdgcn_exp2f(y);
          sum += e;
          ent += e * y;
        }
      sum = over_groups(sum, [](float x, float y) { return x + y; });
      ent = over_groups(ent, [](float x, float y) { return x + y; });
      if (here && grp == 0) {
        a.part[slice] = (floatx2){top, sum};
        a.ent[slice] = ent;
      }
    } else {
      const LpToken k = lp_token(a, row, here, t);
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[nt][i] = lp_grad(k, z[nt][i]);
      if (__ballot(mine) != 0) {
#pragma unroll
        for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) z[nt][i] += at == 4 * nt + i ? k.da : 0.0f;
      }
      // A token without a gradient has none, whatever its logits are.
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[nt][i] = k.none ? 0.0f : fp32_rounded(z[nt][i]);
      // Columns of the piece's last, partial 64 hold zeros: G is read in steps of 64.
      if (mt % 2 == 1) {
        const int64_t first = row0 + 16 * (mt - 1);
        gc_store_bf16<kNT, false>(
            [&](int h, int nt, int i) { return core.acc[mt - 1 + h][nt][i]; },
            lds + 32 * 64 * kNT * wave, a.g + first * a.ldg + r0 + c0, a.ldg, a.M - first,
            a.gcols - (r0 + c0), lane);
      }
    }
  }
}

// Half tiles of one launch: their logits as they are stored.
struct LpSegment {
  int32_t slices, width;
  uint32_t column;   // the first one
  int32_t columns;   // how many there are
  const floatx2 *part;      // [slices][M]
  const float *z;           // [slices][M][width]
};

// G of a piece from kept logits, for half tiles s0 .. of one segment: eight columns a
// lane, kLpKept rows one after the other.  Bound by memory: 6 bytes a logit.
constexpr int kLpKept = 4;
__global__ void __launch_bounds__(256) lp_kept_kernel(const LpLogits a, const LpSegment g,
                                                      int32_t s0, int32_t row_blocks) {
  const int s = s0 + (int)(blockIdx.x / (uint32_t)row_blocks);
  const int eights = g.width / 8, rows = 256 / eights;
  const int o = (int)threadIdx.x % eights;
  const int64_t row0 = (int64_t)(blockIdx.x % (uint32_t)row_blocks) * (rows * kLpKept) +
                       (int)threadIdx.x / eights;
  const int64_t column = (int64_t)g.column + (int64_t)s * g.width + 8 * o;
  if (column - a.v0 >= a.gcols) return;  // G's rows are whole 64s
  floatx4 v[kLpKept][2];
#pragma unroll
  for (int i = 0; i < kLpKept; ++i) {
    const int64_t row = row0 + i * rows;
    if (row >= a.M) break;
    const floatx4 *z =
        reinterpret_cast<const floatx4 *>(g.z + ((int64_t)s * a.M + row) * g.width + 8 * o);
    v[i][0] = __builtin_nontemporal_load(z);
    v[i][1] = __builtin_nontemporal_load(z + 1);
  }
#pragma unroll
  for (int i = 0; i < kLpKept; ++i) {
    const int64_t row = row0 + i * rows;
    if (row >= a.M) break;
    const int64_t t = a.targets[row];
    const LpToken k = lp_token(a, row, true, t);
    const int64_t rel = t - column;
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = lp_grad(k, v[i][j / 4][j % 4]);
      if (t != a.ignore && rel == j && t < a.V) x[j] += k.da;
      x[j] = k.none ? 0.0f : fp32_rounded(x[j]);
    }
    *reinterpret_cast<u32x4 *>(a.g + row * a.ldg + (column - a.v0)) =
        (u32x4){pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]),
                pack_bf16x2(x[6], x[7])};
  }
}

// The largest of a 64-bit key over the wave, in every lane.
template <int kCtrl>
__device__ __forceinline__ uint64_t dpp_max64(uint64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, kCtrl, 0xf, 0xf,
                                                            true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), kCtrl, 0xf,
                                                            0xf, true);
  const uint64_t o = (uint64_t)hi << 32 | lo;
  return o > v ? o : v;
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
  v = dpp_max64<0x128>(v);  // row_ror:8
  v = dpp_max64<0x124>(v);
  v = dpp_max64<0x122>(v);
  v = dpp_max64<0x121>(v);
  const auto l16 = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  const auto h16 =
      __builtin_amdgcn_permlane16_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  uint64_t a = (uint64_t)h16[0] << 32 | l16[0], b = (uint64_t)h16[1] << 32 | l16[1];
  v = a > b ? a : b;
  const auto l32 = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  const auto h32 =
      __builtin_amdgcn_permlane32_swap((uint32_t)(v >> 32), (uint32_t)(v >> 32), false, false);
  a = (uint64_t)h32[0] << 32 | l32[0];
  b = (uint64_t)h32[1] << 32 | l32[1];
  return a > b ? a : b;
}

struct LpSelect {
  LpSegment seg[2];
  int64_t M;
  int32_t k, slices;  // of both segments
  bool first;         // no pieces before
  uint64_t *best;     // [M][k]
};

// Keys a wave ranks at once: two a lane.
constexpr int kLpList = 128;
// Half tiles whose logits are looked at, and those of them at once.
constexpr int kLpHeld = 64, kLpAt = 32;

// Writes visible to the wave's other lanes.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's LDS, in front of the half tiles' maxima.
struct LpWave {
  uint64_t list[kLpList];
  u32x4 lanes[16];  // a value of every lane
  int32_t chosen[kLpHeld];
  uint32_t count[4];
};

// The k-th largest of the lanes' values (0 if fewer have one): below it are none of
// the k largest of all values whose maxima the lanes hold.
__device__ __forceinline__ uint32_t kth_of_lanes(uint32_t v, int k, int lane, LpWave &w) {
  reinterpret_cast<uint32_t *>(w.lanes)[lane] = v;
  wave_lds_fence();
  int ahead = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const u32x4 o = w.lanes[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) ahead += o[j] > v ? 1 : 0;
  }
  // The least of those with fewer than k ahead, as the largest complement.
  uint32_t c = ahead < k ? ~v : 0;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    const uint32_t o = (uint32_t)__shfl_xor((int)c, off, 64);
    c = o > c ? o : c;
  }
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)~c);
}

// The alternatives of a token, by one wave.  Twice the same step, over the half tiles'
// maxima and over the logits of those that are left: the k-th largest of the 64 lanes'
// own maxima is reached by k values at least, so what lies below is out.  What remains,
// about k, is ranked by counting, together with the k best of the pieces before.  Where
// too many are left because they are equal, the first k by their index are enough and
// are taken in that order; where they are not equal (which takes logits sorted against
// the lanes), k rounds over all of them find the k best.
__device__ __forceinline__ void lp_select(const LpSelect &a, int64_t row, int lane, LpWave &w) {
  const int rounds = (a.slices + 63) / 64;
  uint32_t *maxima = reinterpret_cast<uint32_t *>(&w + 1);
  uint64_t *best = a.best + row * a.k;
  const uint64_t before = !a.first && lane < a.k ? best[lane] : 0;
  const uint32_t least = a.first ? 0 : (uint32_t)(best[a.k - 1] >> 32);
  const uint64_t below = (1ull << lane) - 1;
  const LpSegment g0 = a.seg[0], g1 = a.seg[1];
  if (lane < 4) w.count[lane] = 0;

  uint32_t top = 0;
  for (int i0 = 0; i0 < rounds; i0 += 8) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = 64 * (i0 + i) + lane;
      const bool second = s >= g0.slices;
      const floatx2 *p = second ? g1.part + (int64_t)(s - g0.slices) * a.M
                                : g0.part + (int64_t)s * a.M;
      v[i] = s < a.slices ? p[row].x : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int s = 64 * (i0 + i) + lane;
      uint32_t o = s < a.slices ? lp_order(v[i]) : 0;
      // A half tile counts only if its maximum exceeds the k-th best.
      if (o <= least) o = 0;
      if (i0 + i < rounds) maxima[s] = o;
      top = o > top ? o : top;
    }
  }
  if (__ballot(top != 0) == 0) return;  // the pieces before had all
  uint32_t floor = kth_of_lanes(top, a.k, lane, w);
  if (floor == 0) floor = 1;

  // The half tiles that are left.
  int mine = 0;
  for (int i = 0; i < rounds; ++i) mine += maxima[64 * i + lane] >= floor ? 1 : 0;
  if (mine > 0) {
    int at = (int)atomicAdd(&w.count[0], (uint32_t)mine);
    for (int i = 0; i < rounds; ++i)
      if (maxima[64 * i + lane] >= floor) {
        if (at < kLpHeld) w.chosen[at] = 64 * i + lane;
        ++at;
      }
  }
  wave_lds_fence();
  int count = __builtin_amdgcn_readfirstlane((int)w.count[0]);
  // The same by their index, and of those equal to the bound the first k.
  auto pick_in_order = [&] {
    int equal = 0;
    count = 0;
    for (int i = 0; i < rounds; ++i) {
      const uint32_t o = maxima[64 * i + lane];
      const uint64_t same = __ballot(o == floor);
      const bool in = o > floor || (o == floor && equal + __popcll(same & below) < a.k);
      const uint64_t all = __ballot(in);
      const int at = count + __popcll(all & below);
      if (in && at < kLpHeld) w.chosen[at] = 64 * i + lane;
      count += __popcll(all);
      equal += __popcll(same);
    }
    wave_lds_fence();
  };
  const uint32_t bound = floor;  // of the half tiles
  if (count > kLpHeld) pick_in_order();

  // Half tile s: its first column, how many it has, its first logit.
  auto half_tile = [&](int s, uint32_t &column, int &wide, const float *&z) {
    const bool second = s >= g0.slices;
    const int at = second ? s - g0.slices : s, width = second ? g1.width : g0.width;
    const int left = (second ? g1.columns : g0.columns) - at * width;
    column = (second ? g1.column : g0.column) + (uint32_t)(at * width);
    wide = left < width ? left : width;
    z = (second ? g1.z : g0.z) + ((int64_t)at * a.M + row) * width;
  };
  if (count <= kLpHeld) {
    // 32 chosen half tiles from j on, two at a time: a lane has four columns of one.
    struct Logits {
      uint32_t order[kLpAt / 2][4], column[kLpAt / 2];
    };
    auto read = [&](int j, Logits &e) {
      floatx4 v[kLpAt / 2];
      int left[kLpAt / 2];
#pragma unroll
      for (int i = 0; i < kLpAt / 2; ++i) {
        left[i] = 0;
        if (j + 2 * i >= count) continue;
        const int c = j + 2 * i + (lane >> 5);
        const float *z;
        int wide;
        half_tile(w.chosen[c < count ? c : 0], e.column[i], wide, z);
        e.column[i] += 4 * (uint32_t)(lane & 31);
        left[i] = c < count ? wide - 4 * (lane & 31) : 0;
        // (The rows of a half tile are whole, past the last column with -inf.)
        if (left[i] > 0) v[i] = *reinterpret_cast<const floatx4 *>(z + 4 * (lane & 31));
      }
#pragma unroll
      for (int i = 0; i < kLpAt / 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) e.order[i][q] = q < left[i] ? lp_order(v[i][q]) : 0;
    };
    auto most = [&](const Logits &e) {
#pragma unroll
      for (int i = 0; i < kLpAt / 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) top = e.order[i][q] > top ? e.order[i][q] : top;
    };
    Logits e;
    top = 0;
    if (count > kLpAt) {
      read(kLpAt, e);
      most(e);
    }
    read(0, e);
    most(e);
    const uint32_t kth = kth_of_lanes(top, a.k, lane, w);
    floor = kth > floor ? kth : floor;
    // Later columns lose a tie with the pieces before.
    if (floor <= least) floor = least + 1;
    auto gather = [&](const Logits &e) {
      mine = 0;
#pragma unroll
      for (int i = 0; i < kLpAt / 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) mine += e.order[i][q] >= floor ? 1 : 0;
      int at = 0;
      if (mine > 0) at = (int)atomicAdd(&w.count[1], (uint32_t)mine);
#pragma unroll
      for (int i = 0; i < kLpAt / 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const bool in = e.order[i][q] >= floor;
          if (__ballot(in) == 0) continue;
          if (in && at < kLpList) w.list[at] = lp_key(e.order[i][q], e.column[i] + (uint32_t)q);
          at += in ? 1 : 0;
        }
    };
    gather(e);
    if (count > kLpAt) {
      read(kLpAt, e);
      gather(e);
    }
    wave_lds_fence();
    int n = __builtin_amdgcn_readfirstlane((int)w.count[1]);
    const uint64_t had = __ballot(before != 0);
    if (n + __popcll(had) > kLpList) {
      // In the order of the columns, of those equal to the bound the first k.
      const uint32_t f = floor;
      floor = bound;
      pick_in_order();
      floor = f;
      n = 0;
      int equal = 0;
      for (int j = 0; j < count && j < kLpHeld; ++j) {
        uint32_t column;
        int wide;
        const float *z;
        half_tile(__builtin_amdgcn_readfirstlane(w.chosen[j]), column, wide, z);
        for (int c = lane; c < (wide + 63) / 64 * 64; c += 64) {
          const uint32_t o = c < wide ? lp_order(z[c]) : 0;
          const uint64_t same = __ballot(o == floor);
          const bool in = o > floor || (o == floor && equal + __popcll(same & below) < a.k);
          const uint64_t all = __ballot(in);
          const int at = n + __popcll(all & below);
          if (in && at < kLpList) w.list[at] = lp_key(o, column + (uint32_t)c);
          n += __popcll(all);
          equal += __popcll(same);
        }
      }
      if (count > kLpHeld) n = kLpList + 1;
    }
    // The pieces before.
    const int at = n + __popcll(had & below);
    if (before != 0 && at < kLpList) w.list[at] = before;
    n += __popcll(had);
    wave_lds_fence();
    if (n <= kLpList) {
      const uint64_t key[2] = {lane < n ? w.list[lane] : 0,
                               64 + lane < n ? w.list[64 + lane] : 0};
      int ahead[2] = {0, 0};
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const uint64_t o = w.list[i];
        ahead[0] += o > key[0] ? 1 : 0;
        ahead[1] += o > key[1] ? 1 : 0;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (64 * h + lane < n && ahead[h] < a.k) best[ahead[h]] = key[h];
      // (Fewer than k only where the vocabulary's first piece has fewer.)
      if (lane >= n && lane < a.k) best[lane] = 0;
      return;
    }
  }

  uint64_t last = ~0ull;
  for (int t = 0; t < a.k; ++t) {
    uint64_t own = before < last ? before : 0;
    for (int s = 0; s < a.slices; ++s) {
      const uint32_t o = maxima[s];
      if (o == 0 || o < floor) continue;
      uint32_t column;
      int wide;
      const float *z;
      half_tile(s, column, wide, z);
      for (int c = lane; c < wide; c += 64) {
        const uint32_t order = lp_order(z[c]);
        const uint64_t key = order <= least ? 0 : lp_key(order, column + (uint32_t)c);
        if (key < last && key > own) own = key;
      }
    }
    last = wave_max64(own);
    if (lane == 0) best[t] = last;
    if (last == 0) last = 1;
  }
}

// One wave a token.
__global__ void __launch_bounds__(256) lp_select_kernel(const LpSelect a) {
  extern __shared__ __attribute__((aligned(16))) char lp_lds[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 6) + wave;
  if (row >= a.M) return;
  const int bytes = (int)sizeof(LpWave) + (a.slices + 63) / 64 * 256;
  lp_select(a, row, threadIdx.x & 63, *reinterpret_cast<LpWave *>(lp_lds + wave * bytes));
}

struct LpJoin {
  const floatx2 *part;
  const float *ent, *zt;
  const uint64_t *best;
  const int64_t *targets;
  int64_t M;
  int32_t slices, k;
  int64_t V, ignore;
  float *logp, *lse, *entropy, *top_logp;
  int64_t *top_ids;
};

// Maximum, sum of exponentials and sum of e y of some of a token's logits.
struct LpSums {
  float top, sum, ent;
};
__device__ __forceinline__ LpSums lp_none() { return LpSums{-__builtin_inff(), 0.0f, 0.0f}; }
__device__ __forceinline__ LpSums lp_joined(const LpSums &x, const LpSums &y) {
  const float top = fmaxf(x.top, y.top);
  const float ref = top == -__builtin_inff() ? 0.0f : top;
  const float dx = lp_floor((x.top - ref) * kLog2e), dy = lp_floor((y.top - ref) * kLog2e);
  const float ex = __builtin_amdgcn_exp2f(dx), ey = __builtin_amdgcn_exp2f(dy);
  return LpSums{top, x.sum * ex + y.sum * ey,
                (x.ent + dx * x.sum) * ex + (y.ent + dy * y.sum) * ey};
}
// Half tiles first, first + step, .. of a token, four loads ahead.
__device__ __forceinline__ LpSums lp_column(const LpJoin &a, int64_t row, int first, int step) {
  LpSums s = lp_none();
  for (int i = first; i < a.slices; i += 4 * step) {
    LpSums v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = i + j * step;
      v[j] = lp_none();
      if (n < a.slices) {
        const floatx2 p = a.part[(int64_t)n * a.M + row];
        v[j] = LpSums{p.x, p.y, a.ent[(int64_t)n * a.M + row]};
      }
    }
    s = lp_joined(s, lp_joined(lp_joined(v[0], v[1]), lp_joined(v[2], v[3])));
  }
  return s;
}
// A token's results by threads `first`, first + step, .. of the alternatives, the
// first one of which has the rest.
__device__ __forceinline__ void lp_results(const LpJoin &a, int64_t row, const LpSums &s, int first,
                                           int step) {
  const float log_sum = __builtin_amdgcn_logf(s.sum) * kLn2;
  if (first == 0) {
    a.lse[row] = s.top + log_sum;
    a.entropy[row] = log_sum - s.ent / s.sum * kLn2;
    const int64_t t = a.targets[row];
    float v = 0.0f;
    if (t != a.ignore)
      v = t < 0 || t >= a.V ? __builtin_nanf("") : (a.zt[row] - s.top) - log_sum;
    a.logp[row] = v;
  }
  for (int i = first; i < a.k; i += step) {
    const uint64_t key = a.best[row * a.k + i];
    a.top_ids[row * a.k + i] = (int64_t)(uint32_t)~(uint32_t)key;
    a.top_logp[row * a.k + i] = (lp_value((uint32_t)(key >> 32)) - s.top) - log_sum;
  }
}

// Joins a token's partial sums: 32 threads a token take every 32nd half tile, then
// meet in a fixed order.
constexpr int kLpTokens = 8;
__global__ void __launch_bounds__(256) lp_join_kernel(const LpJoin a) {
  constexpr int kGroups = 256 / kLpTokens;
  __shared__ LpSums lds[kGroups][kLpTokens];
  const int tok = threadIdx.x % kLpTokens, grp = threadIdx.x / kLpTokens;
  const int64_t row = (int64_t)blockIdx.x * kLpTokens + tok;
  lds[grp][tok] = row < a.M ? lp_column(a, row, grp, kGroups) : lp_none();
#pragma unroll
  for (int half = kGroups / 2; half >= 1; half /= 2) {
    __syncthreads();
    if (grp < half) lds[grp][tok] = lp_joined(lds[grp][tok], lds[grp + half][tok]);
  }
  __syncthreads();
  if (row < a.M) lp_results(a, row, lds[0][tok], grp, kGroups);
}

// Few tokens: a workgroup a token, whose first wave finds the alternatives of the last
// piece while the others join the sums.
__global__ void __launch_bounds__(256) lp_finish_kernel(const LpSelect c, const LpJoin a) {
  extern __shared__ __attribute__((aligned(16))) char lp_lds[];
  __shared__ LpSums lds[3];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x;
  if (wave == 0) {
    if (a.k > 0) lp_select(c, row, lane, *reinterpret_cast<LpWave *>(lp_lds));
  } else {
    LpSums s = lp_column(a, row, threadIdx.x - 64, 192);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1)
      s = lp_joined(s, LpSums{__shfl_xor(s.top, off, 64), __shfl_xor(s.sum, off, 64),
                              __shfl_xor(s.ent, off, 64)});
    if (lane == 0) lds[wave - 1] = s;
  }
  __syncthreads();
  if (wave == 0) lp_results(a, row, lp_joined(lp_joined(lds[0], lds[1]), lds[2]), lane, 64);
}

// C = max |dlogp| over the tokens that have one, or max |dentropy| if that is 2^64 times
// as large (G would leave fp32's range), or 1.
__global__ void __launch_bounds__(1024) lp_common_kernel(const float *dlogp, const float *dentropy,
                                                         const int64_t *targets, int64_t ignore,
                                                         int64_t M, float *common) {
  __shared__ float part[2][16];
  float top[2] = {0.0f, 0.0f};
  // A NaN counts as infinite: fmaxf would drop it.
  auto size = [](float v) { return fabsf(v) < __builtin_inff() ? fabsf(v) : __builtin_inff(); };
  for (int64_t i = threadIdx.x; i < M; i += 1024) {
    if (targets[i] != ignore) top[0] = fmaxf(top[0], size(dlogp[i]));
    if (dentropy != nullptr) top[1] = fmaxf(top[1], size(dentropy[i]));
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top[j] = fmaxf(top[j], __shfl_xor(top[j], off, 64));
    if ((threadIdx.x & 63) == 0) part[j][threadIdx.x >> 6] = top[j];
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int j = 0; j < 2; ++j)
    for (int i = 1; i < 16; ++i) top[j] = fmaxf(top[j], part[j][i]);
  const float c = top[0] > 0.0f && top[1] <= top[0] * 0x1p64f ? top[0] : top[1];
  *common = c == 0.0f || c == __builtin_inff() ? 1.0f : c;
}

// Launches over the logits: those of the cross entropy, but tiles of 64 x 64, which have
// more loads in flight, in two cases.  Where each is alone on a CU, a CU's share being
// half of what it is in tiles of 64 x 128: whole calls of one token, 8000 columns of 8192
// 66 -> 39 us, of 2048 20.5 -> 18.5, 16000 of 4096 40 -> 30; of 64 tokens 43 -> 33; what
// whole rounds leave of 1000 tokens, 50021 of 5120, 470 -> 456 (with alternatives).  And
// where two of them fill at least three quarters of the CUs' places, and few tokens
// leave the rows of x out: one token, 32000 of 4096 58.7 -> 51.8, 28000 of 4096 53 -> 46.
// (Half full, 17000 of 8192, 73 would become 82; 64 tokens, 28000 of 8192, 93 98.)  A
// call of more tiles than there are places keeps the larger ones, however full its last
// round of small ones would be; what whole rounds leave is a launch like any other.
static int lp_tiles(int64_t m, int64_t v, int64_t d, CeLaunch (&l)[2]) {
  const int n = ce_tiles(m, v, d, l);
  const int64_t slots = cu_slots();
  for (int i = 0; i < n; ++i) {
    if (l[i].mt != 1) continue;
    const int64_t tiles = ceil_to(m, 64) * ceil_to(l[i].cols, 64);
    if (tiles <= slots || (m <= 32 && d >= 2048 && 2 * tiles >= 3 * slots && tiles <= 2 * slots))
      l[i].nt = 1;
  }
  return n;
}
static int64_t lp_slices(const CeLaunch &l) { return 2 * ceil_to(l.cols, 64 * l.nt); }

// Where the forward of M tokens keeps what.
struct LpLayout {
  int64_t piece;   // columns of a piece of the vocabulary
  int64_t slices;  // partial sums of a token
  int64_t ent, zt, best, z, bytes;
};

static LpLayout lp_layout(int64_t M, int64_t v, int64_t d, int64_t k) {
  LpLayout l{};
  l.piece = v;
  if (k > 0) {
    // Whole rounds of 256 x 256 tiles, as far as they fit.
    int64_t cols = kLpPieceBytes / (4 * M);
    if (cols > kLpPieceCols) cols = kLpPieceCols;
    const int64_t tl = ceil_to(M, 256), round = cu_slots() > tl ? cu_slots() / tl * 256 : 256;
    cols = cols >= round ? cols / round * round : cols / 256 * 256;
    if (cols < 4096) cols = 4096;
    if (cols < v) l.piece = cols;
  }
  int64_t z = 0;
  for (int64_t v0 = 0; v0 < v; v0 += l.piece) {
    const int64_t vn = v - v0 < l.piece ? v - v0 : l.piece;
    // Whole pieces are alike.
    const int64_t n = vn == l.piece ? v / l.piece : 1;
    CeLaunch t[2];
    int64_t cols = 0;
    const int launches = lp_tiles(M, vn, d, t);
    for (int i = 0; i < launches; ++i) {
      l.slices += n * lp_slices(t[i]);
      cols += up(t[i].cols, 64 * t[i].nt);
    }
    if (cols > z) z = cols;
    v0 += (n - 1) * l.piece;
  }
  int64_t at = up(l.slices * M * 8, 256);
  auto take = [&](int64_t n) {
    const int64_t from = at;
    at += up(n, 256);
    return from;
  };
  l.ent = take(l.slices * M * 4);
  l.zt = take(M * 4);
  l.best = take(M * k * 8);
  l.z = take(k > 0 ? z * M * 4 : 0);
  l.bytes = at;
  return l;
}

static int64_t lp_forward_bytes(const CePlan &p, int64_t m, int64_t v, int64_t d, int64_t k) {
  if (m == 0) return 0;
  int64_t bytes = lp_layout(p.tokens, v, d, k).bytes;
  if (m % p.tokens != 0) {
    const int64_t last = lp_layout(m % p.tokens, v, d, k).bytes;
    if (last > bytes) bytes = last;
  }
  return bytes;
}

static int32_t lp_plan(int64_t m, int64_t v, int64_t d, int64_t k, CePlan &p) {
  const int32_t rc = ce_plan(m, v, d, p);
  if (rc != NF4S_OK) return rc;
  if (k < 0) return fail(NF4S_ERR_INVALID_ARGUMENT, "negative number of alternatives");
  if (k > kLpTop || k > v)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "%lld alternatives of %lld tokens: at most %d",
                (long long)k, (long long)v, kLpTop);
  return NF4S_OK;
}

// The logits of a.M tokens and a.vn columns, in one launch or two; with `seg` the
// launches' half tiles.
template <bool kGrad>
static int32_t lp_logits(LpLogits a, int64_t *slices, LpSegment *seg, hipStream_t s) {
  CeLaunch l[2];
  const int n = lp_tiles(a.M, a.vn, a.d, l);
  int64_t done = 0;
  for (int i = 0; i < n; ++i) {
    a.vn = (int32_t)l[i].cols;
    a.tiles_l = (int32_t)ceil_to(a.M, 64 * l[i].mt);
    a.tiles_r = (int32_t)ceil_to(a.vn, 64 * l[i].nt);
    auto *kernel = l[i].mt == 4   ? lp_logits_kernel<4, 4, kGrad>
                   : l[i].mt == 2 ? lp_logits_kernel<2, 4, kGrad>
                   : l[i].nt == 2 ? lp_logits_kernel<1, 2, kGrad>
                                  : lp_logits_kernel<1, 1, kGrad>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)a.tiles_l * (uint32_t)a.tiles_r), dim3(kGcThreads),
                       0, s, a);
    const int32_t rc = check_launch("lp_logits_kernel");
    if (rc != NF4S_OK) return rc;
    if (seg != nullptr)
      seg[i] = LpSegment{2 * a.tiles_r, 32 * l[i].nt, (uint32_t)a.v0, a.vn, a.part, a.z};
    a.w += a.vn * a.d;
    a.v0 += a.vn;
    if (kGrad) {
      a.g += a.vn;
      a.gcols -= a.vn;
    } else {
      a.part += 2 * a.tiles_r * a.M;
      a.ent += 2 * a.tiles_r * a.M;
      if (a.z != nullptr) a.z += (int64_t)a.tiles_r * (64 * l[i].nt) * a.M;
    }
    done += 2 * a.tiles_r;
  }
  if (slices != nullptr) *slices = done;
  return NF4S_OK;
}

// Where kept logits lie: the half tiles of the launches over all columns.
static int64_t lp_kept(int64_t m, int64_t v, int64_t d, const float *z, LpSegment (&seg)[2]) {
  CeLaunch l[2];
  const int n = lp_tiles(m, v, d, l);
  int64_t at = 0, column = 0;
  seg[1] = LpSegment{};
  for (int i = 0; i < n; ++i) {
    const int64_t slices = lp_slices(l[i]), width = 32 * l[i].nt;
    seg[i] = LpSegment{(int32_t)slices, (int32_t)width, (uint32_t)column, (int32_t)l[i].cols,
                       nullptr, z != nullptr ? z + at * m : nullptr};
    at += slices * width;
    column += l[i].cols;
  }
  return at * m * 4;
}

struct LpGrad {
  LpLogits a;
  bool kept;
  LpSegment seg[2];
};

static int32_t lp_grad_logits(const void *ctx, const HeadPiece &p) {
  const LpGrad &c = *static_cast<const LpGrad *>(ctx);
  LpLogits a = c.a;
  a.w += p.v0 * a.d;
  a.v0 = p.v0;
  a.vn = (int32_t)p.vn;
  a.common = p.common;
  a.g = p.g;
  a.ldg = a.gcols = p.ldg;
  if (!c.kept) return lp_logits<true>(a, nullptr, nullptr, p.stream);
  // Pieces begin at multiples of 256 columns and launches too, so at half tiles.
  for (int i = 0; i < 2; ++i) {
    const LpSegment &g = c.seg[i];
    const int64_t end = (int64_t)g.column + g.columns;
    const int64_t from = p.v0 > g.column ? p.v0 : g.column;
    const int64_t to = p.v0 + p.vn < end ? p.v0 + p.vn : end;
    if (g.slices == 0 || from >= to) continue;
    // Whole 64s, as G's rows: of 32 columns the vocabulary's last half tile may be none.
    const int64_t s0 = (from - g.column) / g.width;
    const int64_t s1 = ceil_to(up(to - g.column, 64), g.width);
    const int64_t blocks = ceil_to(a.M, 256 / (g.width / 8) * kLpKept);
    hipLaunchKernelGGL(lp_kept_kernel, dim3((uint32_t)((s1 - s0) * blocks)), dim3(256), 0,
                       p.stream, a, g, (int32_t)s0, (int32_t)blocks);
    const int32_t rc = check_launch("lp_kept_kernel");
    if (rc != NF4S_OK) return rc;
  }
  return NF4S_OK;
}

}  // namespace nf4s

using namespace nf4s;

extern "C" {

int32_t nf4s_linear_logprob_workspace_size(int64_t m, int64_t v, int64_t d, int64_t top_k,
                                           int32_t backward, int64_t *bytes) {
  clear_error();
  if (bytes == nullptr) return fail(NF4S_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = 0;
  CePlan p;
  const int32_t rc = lp_plan(m, v, d, top_k, p);
  if (rc == NF4S_OK && m > 0)
    *bytes = backward ? p.bwd_bytes : lp_forward_bytes(p, m, v, d, top_k);
  return rc;
}

int32_t nf4s_linear_logprob_logits_size(int64_t m, int64_t v, int64_t d, int64_t *bytes) {
  clear_error();
  if (bytes == nullptr) return fail(NF4S_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = 0;
  CePlan p;
  const int32_t rc = lp_plan(m, v, d, 0, p);
  LpSegment seg[2];
  if (rc == NF4S_OK && m > 0 && m == p.tokens) *bytes = lp_kept(m, v, d, nullptr, seg);
  return rc;
}

int32_t nf4s_linear_logprob_fwd(const uint16_t *x, const uint16_t *w, const int64_t *targets,
                                int64_t m, int64_t v, int64_t d, int64_t top_k,
                                int64_t ignore_index, float *logp, float *lse, float *entropy,
                                float *top_logp, int64_t *top_ids, float *logits, void *workspace,
                                int64_t workspace_bytes, void *stream) {
  clear_error();
  CePlan p;
  int32_t rc = lp_plan(m, v, d, top_k, p);
  if (rc != NF4S_OK || m == 0) return rc;
  rc = ce_operands(x, w, targets, m, workspace, workspace_bytes,
                   lp_forward_bytes(p, m, v, d, top_k));
  if (rc != NF4S_OK) return rc;
  if (logp == nullptr || lse == nullptr || entropy == nullptr ||
      (top_k > 0 && (top_logp == nullptr || top_ids == nullptr)))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "an output is NULL");
  if (!aligned(logp, 4) || !aligned(lse, 4) || !aligned(entropy, 4) || !aligned(top_logp, 4) ||
      !aligned(top_ids, 8) || !aligned(logits, 16))
    return fail(NF4S_ERR_MISALIGNED,
                "outputs must be aligned to their elements, logits 16-byte");
  if (logits != nullptr && (top_k > 0 || m != p.tokens))
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE,
                "logits are kept of up to %lld tokens, without alternatives",
                (long long)kCeTokens);
  const hipStream_t s = as_stream(stream);
  char *base = static_cast<char *>(workspace);
  for (int64_t m0 = 0; m0 < m; m0 += p.tokens) {
    LpLogits a{};
    a.M = m - m0 < p.tokens ? m - m0 : p.tokens;
    const LpLayout l = lp_layout(a.M, v, d, top_k);
    uint64_t *best = reinterpret_cast<uint64_t *>(base + l.best);
    a.x = x + m0 * d;
    a.targets = targets + m0;
    a.d = d;
    a.V = v;
    a.ignore = ignore_index;
    a.k = (int32_t)top_k;
    a.part = reinterpret_cast<floatx2 *>(base);
    a.ent = reinterpret_cast<float *>(base + l.ent);
    a.zt = reinterpret_cast<float *>(base + l.zt);
    a.z = top_k > 0 ? reinterpret_cast<float *>(base + l.z) : logits;
    const bool few = a.M < 512;
    LpSelect sel{};
    int64_t lds = 0;
    for (int64_t v0 = 0; v0 < v; v0 += l.piece) {
      a.w = w + v0 * d;
      a.v0 = v0;
      a.vn = (int32_t)(v - v0 < l.piece ? v - v0 : l.piece);
      a.best = v0 > 0 && top_k > 0 ? best : nullptr;
      int64_t slices = 0;
      rc = lp_logits<false>(a, &slices, sel.seg, s);
      if (rc != NF4S_OK) return rc;
      if (top_k > 0) {
        sel.M = a.M;
        sel.k = (int32_t)top_k;
        sel.slices = (int32_t)slices;
        sel.first = v0 == 0;
        sel.best = best;
        lds = (int64_t)sizeof(LpWave) + (slices + 63) / 64 * 256;
        if (!few || v0 + l.piece < v) {
          const int64_t fit = kLpSelectLds / lds, waves = fit < 4 ? fit : 4;
          hipLaunchKernelGGL(lp_select_kernel, dim3((uint32_t)ceil_to(a.M, waves)),
                             dim3((uint32_t)(64 * waves)), (uint32_t)(waves * lds), s, sel);
          rc = check_launch("lp_select_kernel");
          if (rc != NF4S_OK) return rc;
        }
      }
      a.part += slices * a.M;
      a.ent += slices * a.M;
    }
    LpJoin j{};
    j.part = reinterpret_cast<floatx2 *>(base);
    j.ent = reinterpret_cast<float *>(base + l.ent);
    j.zt = a.zt;
    j.best = best;
    j.targets = a.targets;
    j.M = a.M;
    j.slices = (int32_t)l.slices;
    j.k = (int32_t)top_k;
    j.V = v;
    j.ignore = ignore_index;
    j.logp = logp + m0;
    j.lse = lse + m0;
    j.entropy = entropy + m0;
    j.top_logp = top_k > 0 ? top_logp + m0 * top_k : nullptr;
    j.top_ids = top_k > 0 ? top_ids + m0 * top_k : nullptr;
    if (few)
      hipLaunchKernelGGL(lp_finish_kernel, dim3((uint32_t)a.M), dim3(256), (uint32_t)lds, s, sel,
                         j);
    else
      hipLaunchKernelGGL(lp_join_kernel, dim3((uint32_t)ceil_to(a.M, kLpTokens)), dim3(256), 0, s,
                         j);
    rc = check_launch("lp_join_kernel");
    if (rc != NF4S_OK) return rc;
  }
  return NF4S_OK;
}

int32_t nf4s_linear_logprob_bwd(const uint16_t *x, const uint16_t *w, const int64_t *targets,
                                const float *lse, const float *entropy, const float *logits,
                                const float *dlogp, const float *dentropy, int64_t m, int64_t v,
                                int64_t d, int64_t ignore_index, uint16_t *dx, void *dw,
                                int32_t dw_is_f32, int32_t accumulate, void *workspace,
                                int64_t workspace_bytes, void *stream) {
  clear_error();
  CePlan p;
  int32_t rc = lp_plan(m, v, d, 0, p);
  if (rc != NF4S_OK) return rc;
  rc = ce_operands(x, w, targets, m, workspace, workspace_bytes, p.bwd_bytes);
  if (rc != NF4S_OK) return rc;
  if (accumulate && !dw_is_f32)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "dw accumulates in fp32 only");
  if (dw == nullptr || (m > 0 && (lse == nullptr || dlogp == nullptr || dx == nullptr)))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "lse, dlogp, dx or dw is NULL");
  if (m > 0 && dentropy != nullptr && entropy == nullptr)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "dentropy needs entropy");
  if (logits != nullptr && m > 0 && m != p.tokens)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "logits are kept of up to %lld tokens",
                (long long)kCeTokens);
  if (!aligned(dw, 16) || (m > 0 && (!aligned(dx, 16) || !aligned(lse, 4) || !aligned(dlogp, 4) ||
                                     !aligned(entropy, 4) || !aligned(dentropy, 4) ||
                                     !aligned(logits, 16))))
    return fail(NF4S_ERR_MISALIGNED,
                "dx, dw and logits must be 16-byte aligned, the tokens' values 4-byte");
  const hipStream_t s = as_stream(stream);
  if (m == 0) return accumulate ? NF4S_OK : head_zero_dw(dw, dw_is_f32 != 0, v * d, s);
  const HeadGrad h{x, w, m, v, d, dx, dw, dw_is_f32 != 0, accumulate != 0, workspace};
  hipLaunchKernelGGL(lp_common_kernel, dim3(1), dim3(1024), 0, s, dlogp, dentropy, targets,
                     ignore_index, m, head_common(h, p));
  rc = check_launch("lp_common_kernel");
  if (rc != NF4S_OK) return rc;
  LpGrad c{};
  LpLogits &a = c.a;
  a.x = x;
  a.w = w;
  a.targets = targets;
  a.M = m;
  a.d = d;
  a.V = v;
  a.ignore = ignore_index;
  a.lse = lse;
  a.entropy = entropy;
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  c.kept = logits != nullptr;
  if (c.kept) lp_kept(m, v, d, logits, c.seg);
  return head_gradients(h, p, lp_grad_logits, &c, s);
}

}  // extern "C"
