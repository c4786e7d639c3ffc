// linear_ce.hip - cross entropy of a linear head over a large vocabulary, with
// its gradients, without keeping the logits, for gfx950 (MI355X).
//
// x [M, d] and w [V, d] bf16, one target a token (the reference streams the
// vocabulary in tiles with an online softmax, doublepass/src/loss.rs and
// doublepass/kernels/fused_ce.cu:71-173):
//   z = x . w^T,  lse_m = log sum_c exp z_mc,  loss_m = lse_m - z_m,t(m)
//   G_mc = (exp(z_mc - lse_m) - [c = t(m)]) dloss_m / c
//   dx = c G . w,   dw = c G^T . x,   c = max |dloss|
// An ignored target gives loss 0 and a row of G that is 0 (times its row of x in
// dw: what is not finite there reaches dw); one outside [0, V) that is not the
// ignored value gives NaN.  Products accumulate in fp32; maxima, sums, lse and
// loss are fp32.
//
// Forward: a tile of logits (tokens x vocabulary) stays in its accumulators; a
// lane holds one token's columns, so the tile's maximum and sum of exponentials
// are sums over registers and one exchange.  They leave as 8 bytes per token
// and 32 kNT columns, and a second kernel joins them: M V / 16 bytes written at
// 256 x 256 tiles, where the logits would be 2 M V.
// Backward: the vocabulary in pieces whose G (bf16, the operand of both
// products: one rounding of each value, as of every dY of the weight gradients)
// fits kCePieceBytes.  G in two bf16 terms would double two of the four products.
// The common factor c stays out of G: the tokens of a mean all have dloss = c,
// whose rounding error would be that of every target's entry (up to 2^-8 at once);
// divided by c those entries are close to -1.  What the rounding costs, relative
// errors of 77 to 512 tokens over 4000 to 32000 columns: of a mean, dx and the
// rows of dw that are some token's target 0.0017, as a bf16 result alone; the
// other rows of dw 0.0023; in an fp32 dw 0.0001 and 0.0016.  With a weight for each
// token its target's entry is rounded like any other: dx and the targets' rows
// 0.0022, in an fp32 dw 0.0013.  Per piece: logits again, turned into G in the
// epilogue; dx += G . w in fp32; the piece's rows of dw.
//
// Measured at 4096 tokens, 128000 x 8192: forward 5.95 ms (1443 TFLOP/s), a piece
// of 32000 columns 1627 us for G (1320), 1519 for dx (1414), 1576 for dw (1363);
// library products of these shapes run at 1490, 1328 and 1147.  The matrix
// pipe is busy 65-72 % of the cycles, at a clock that has fallen to 1.77-1.91
// GHz: power sets the rate (bf16_gemm_core.hpp), and waves wait 13-18 % of their
// time.  Few tokens read w once for each product and write dw: one token over
// 128000 x 8192, gradients 1142 us (5.5 TB/s), forward 363 us (5.8).  dw in fp32
// instead of bf16, stored and accumulated: 1486 and 2908 us there; 224 and 401
// for 77 tokens, 32000 x 4096 (bf16 202); 18.9 and 20.7 ms for 4096 tokens, 128000
// x 8192 (18.6).
#include <cmath>

#include "bf16_gemm_core.hpp"

namespace nf4s {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// G of a piece: what the Infinity Cache (256 MB) holds between the kernel that
// writes it and the two that read it.  Gradients of 8192 x 32000 x 4096: 4813 us
// with 256 MB, 4941 with half, 4772 with four times as much; of 4096 x 128000 x
// 8192 18.9, 19.1 and 18.6 ms.
constexpr int64_t kCePieceBytes = (int64_t)256 << 20;
// Tokens of one forward launch, which bounds its partial sums.
constexpr int64_t kCeTokens = 16384;
// A launch counts its threads in 32 bits.
constexpr int64_t kMaxTiles = 0xffffffffll / kGcThreads;

// Maximum and sum of exponentials of part of a token's logits.
typedef float floatx2 __attribute__((ext_vector_type(2)));

struct CeLogits {
  const uint16_t *x, *w;  // w at the piece's first row
  const int64_t *targets;
  int64_t M, d;
  int64_t v0;        // first column of the piece
  int32_t vn;        // its columns
  int64_t V, ignore;
  int32_t tiles_l, tiles_r, strip;
  // forward
  floatx2 *part;     // [2 tiles_r][M]
  float *zt;         // [M] logit of the target
  // backward
  const float *lse, *dloss;
  const float *common;  // c
  uint16_t *g;       // [M, ldg]
  int64_t ldg, gcols;  // row length of G, columns of it from g on
};

// The largest, or the sum, over the four lanes l % 16 + 16 g that hold a token's
// columns, in each of them.
template <class F>
__device__ __forceinline__ float over_groups(float v, F &&f) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  v = f(__builtin_bit_cast(float, (uint32_t)s[0]), __builtin_bit_cast(float, (uint32_t)s[1]));
  const uint32_t c = __builtin_bit_cast(uint32_t, v);
  const auto t = __builtin_amdgcn_permlane32_swap(c, c, false, false);
  return f(__builtin_bit_cast(float, (uint32_t)t[0]), __builtin_bit_cast(float, (uint32_t)t[1]));
}

__device__ __forceinline__ float exp_of(float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}

// Column of the wave's block (0 .. 32 kNT - 1) of the lane's register i of column
// tile nt is 16 nt + 4 (lane / 16) + i, its token of row tile mt 16 mt + lane % 16.
template <int kMT, int kNT, bool kGrad>
__global__ void __launch_bounds__(kGcThreads, kMT == 1 ? 2 : 1) ce_logits_kernel(const CeLogits a) {
  using Core = GcCore<kMT, kNT, false, false>;
  __shared__ __attribute__((aligned(16))) char lds[Core::kLdsBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  int tl, tr;
  gc_tile(blockIdx.x, a.tiles_l, a.tiles_r, a.strip, tl, tr);
  const int64_t l0 = (int64_t)tl * Core::kTileL;
  const int r0 = tr * Core::kTileR;
  const int64_t lrows = a.M - l0 < Core::kTileL ? a.M - l0 : Core::kTileL;
  const int rrows = a.vn - r0 < Core::kTileR ? a.vn - r0 : Core::kTileR;
  Core core;
  core.run(gc_along(a.x + l0 * a.d, a.d, lrows, a.d),
           gc_along(a.w + (int64_t)r0 * a.d, a.d, rrows, a.d), a.d, lds, lane, wave);

  const int64_t row0 = l0 + 32 * kMT * (wave >> 1);  // the wave's first token
  const int c0 = 32 * kNT * (wave & 1);              // and its first column in the tile
  const int cols = rrows - c0;                       // its columns that exist (may be <= 0)
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
      // Nothing but -inf: any finite reference gives a sum of 0.
      const float ref = top == -__builtin_inff() ? 0.0f : top;
      float sum = 0.0f;
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += exp_of(z[nt][i] - ref);
      sum = over_groups(sum, [](float x, float y) { return x + y; });
      if (here && grp == 0)
        a.part[(int64_t)(2 * tr + (wave & 1)) * a.M + row] = (floatx2){top, sum};
    } else {
      const float lse = here ? a.lse[row] : 0.0f;
      const bool skip = t == a.ignore;
      float dl = here && !skip ? a.dloss[row] / *a.common : 0.0f;
      if (!skip && (t < 0 || t >= a.V)) dl = __builtin_nanf("");
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[nt][i] = exp_of(z[nt][i] - lse);
      if (__ballot(mine) != 0) {
#pragma unroll
        for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) z[nt][i] -= at == 4 * nt + i ? 1.0f : 0.0f;
      }
#pragma unroll
      for (int nt = 0; nt < 2 * kNT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) z[nt][i] = skip ? 0.0f : fp32_rounded(z[nt][i] * dl);
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

// Joins a token's partial sums: 256 / kTokens threads a token take every so many
// slices, four loads ahead, then meet in a fixed order.
template <int kTokens>
__global__ void __launch_bounds__(256) ce_join_kernel(const floatx2 *part, const float *zt,
                                                      const int64_t *targets, int64_t M,
                                                      int32_t slices, int64_t V, int64_t ignore,
                                                      float *loss, float *lse) {
  constexpr int kGroups = 256 / kTokens;
  __shared__ floatx2 lds[kGroups][kTokens];
  const int tok = threadIdx.x % kTokens, grp = threadIdx.x / kTokens;
  const int64_t row = (int64_t)blockIdx.x * kTokens + tok;
  auto join = [](floatx2 a, floatx2 b) {
    const float top = fmaxf(a.x, b.x);
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    return (floatx2){top, a.y * exp_of(a.x - ref) + b.y * exp_of(b.x - ref)};
  };
  const floatx2 none = {-__builtin_inff(), 0.0f};
  floatx2 s = none;
  if (row < M)
    for (int i = grp; i < slices; i += 4 * kGroups) {
      floatx2 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = i + j * kGroups;
        v[j] = n < slices ? part[(int64_t)n * M + row] : none;
      }
      s = join(s, join(join(v[0], v[1]), join(v[2], v[3])));
    }
  lds[grp][tok] = s;
#pragma unroll
  for (int half = kGroups / 2; half >= 1; half /= 2) {
    __syncthreads();
    if (grp < half) lds[grp][tok] = join(lds[grp][tok], lds[grp + half][tok]);
  }
  if (grp != 0 || row >= M) return;
  s = lds[0][tok];
  const float l = s.x + __builtin_amdgcn_logf(s.y) * kLn2;
  lse[row] = l;
  const int64_t t = targets[row];
  float v = 0.0f;
  if (t != ignore)
    v = t < 0 || t >= V ? __builtin_nanf("")
                        : (s.x - zt[row]) + __builtin_amdgcn_logf(s.y) * kLn2;
  loss[row] = v;
}

struct CeProduct {
  const uint16_t *l, *r;
  int64_t ldl, ldr;
  int64_t rows, cols;   // of the output
  int64_t k;            // reduction
  int64_t slice;        // reduction of one slice (a multiple of kGcStep)
  int32_t tiles_l, tiles_r, strip;
  void *out;            // leading dimension ld
  int64_t ld, slice_stride;
  const float *common;  // dw: the factor of the products
};

// Output of a product: dx partials (fp32, stored or added) along the vocabulary,
// dw (fp32 or bf16) along the tokens.  dw is not read again and leaves by
// non-temporal stores: 77 tokens, 32000 x 4096, gradients 236 -> 207 us.
enum { kOutF32, kOutF32Add, kOutBf16 };

template <int kMT, int kNT, bool kLAcross, int kOut>
__global__ void __launch_bounds__(kGcThreads, kMT * kNT == 4 ? 2 : 1) ce_product_kernel(
    const CeProduct a) {
  using Core = GcCore<kMT, kNT, kLAcross, true>;
  __shared__ __attribute__((aligned(16))) char lds[Core::kLdsBytes];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int T = a.tiles_l * a.tiles_r;
  const int slice = (int)blockIdx.x / T;
  int tl, tr;
  gc_tile((int)blockIdx.x - slice * T, a.tiles_l, a.tiles_r, a.strip, tl, tr);
  const int64_t l0 = (int64_t)tl * Core::kTileL, r0 = (int64_t)tr * Core::kTileR;
  const int64_t k0 = slice * a.slice;
  const int64_t k = a.k - k0 < a.slice ? a.k - k0 : a.slice;
  const GcOperand r = gc_across(a.r + k0 * a.ldr + r0, a.ldr, a.cols - r0, k);
  Core core;
  if constexpr (kLAcross) {
    // G's rows are ldl long: the zeros past the piece's columns are there too.
    core.run(gc_across(a.l + k0 * a.ldl + l0, a.ldl, a.ldl - l0, k), r, k, lds, lane, wave);
  } else {
    const int64_t rows = a.rows - l0 < Core::kTileL ? a.rows - l0 : Core::kTileL;
    core.run(gc_along(a.l + l0 * a.ldl + k0, a.ldl, rows, (k + 7) & ~(int64_t)7), r, k, lds, lane,
             wave);
  }
  const int64_t row0 = 32 * kMT * (wave >> 1), c0 = r0 + 32 * kNT * (wave & 1);
  const float common = kLAcross ? *a.common : 1.0f;
#pragma unroll
  for (int mt = 0; mt < kMT; ++mt) {
    auto value = [&](int h, int nt, int i) {
      const float v = core.acc[2 * mt + h][nt][i];
      return kLAcross ? fp32_rounded(v * common) : v;
    };
    const int64_t row = l0 + row0 + 32 * mt;
    const int64_t at = slice * a.slice_stride + row * a.ld + c0;
    if constexpr (kOut == kOutBf16)
      gc_store_bf16<kNT, true>(value, lds + 2048 * kNT * wave,
                               static_cast<uint16_t *>(a.out) + at, a.ld, a.rows - row,
                               a.cols - c0, lane);
    else
      gc_store_f32<kNT, kOut == kOutF32Add, kLAcross>(
          value, lds + 4096 * kNT * wave, static_cast<float *>(a.out) + at, a.ld, a.rows - row,
          a.cols - c0, lane);
  }
}

// dx = c times the sum of its slices' fp32 sums, rounded once.
__global__ void __launch_bounds__(256) ce_dx_kernel(const floatx4 *part, int32_t slices,
                                                    int64_t chunks, const float *common,
                                                    u32x2 *dx) {
  const float c = *common;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < chunks;
       i += (int64_t)gridDim.x * 256) {
    floatx4 s = part[i];
    for (int p = 1; p < slices; ++p) s += part[p * chunks + i];
    dx[i] = (u32x2){pack_bf16x2(fp32_rounded(s[0] * c), fp32_rounded(s[1] * c)),
                    pack_bf16x2(fp32_rounded(s[2] * c), fp32_rounded(s[3] * c))};
  }
}

// c = max |dloss|, or 1 if that is zero or not finite.
__global__ void __launch_bounds__(1024) ce_common_kernel(const float *dloss,
                                                         const int64_t *targets, int64_t ignore,
                                                         int64_t M, float *common) {
  __shared__ float part[16];
  float top = 0.0f;
  for (int64_t i = threadIdx.x; i < M; i += 1024) {
    // A NaN counts as infinite (fmaxf would drop it); an ignored token not at all.
    const float v = fabsf(dloss[i]);
    if (targets[i] != ignore) top = fmaxf(top, v < __builtin_inff() ? v : __builtin_inff());
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x != 0) return;
  for (int i = 1; i < 16; ++i) top = fmaxf(top, part[i]);
  *common = top == 0.0f || top == __builtin_inff() ? 1.0f : top;
}

template <typename T>
__global__ void ce_zero_kernel(T *p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    p[i] = T(0);
}

constexpr int64_t kCeFewTokens = 128;

// Tile columns of a strip (gc_tile): 4096 x 32000 x 8192 forward 1520 us with 4,
// 1549 with 6, 1577 with 8, 1666 with 16.
constexpr int kCeStrip = 4;

static int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// A logits launch: 64 mt x 64 nt tiles over the next `cols` columns.
struct CeLaunch {
  int mt, nt;
  int64_t cols;
};

// The tiles of m > 0 tokens by v > 0 columns of length d, as one launch, or as
// whole rounds of large tiles and the rest in smaller ones.  Cost of a launch in
// us: each round takes, per step of 64, `lo` when few tiles run to `hi` when the
// chip is full (less traffic and a higher clock when it is not); w is read at
// `tbs`, again by part for each further row of tiles; 8 us beside for each launch.
// Fitted to all choices at 615 forwards of 1 to 2000 tokens over 1000 to 150000
// columns, d = 512 to 8192, and 54 gradients, with w from memory (in turn from
// copies that no cache holds together): 0.2 % from the best on average, within
// 2 % at 645 of them, 10 % at most.  Times in us at d = 4096 with 64 x 128, 128 x
// 256 and 256 x 256 tiles:
//   1 token, 32000 columns 61, 66, 98;  50021 columns 80, 91, 109;
//   77 tokens, 32000 columns 66, 69, 100;  50021 columns 111, 92, 110;
//   128 tokens, 32000 columns 71, 70, 100;  256 tokens 115, 72, 100;
//   512 tokens 204, 122, 107;
//   1000 tokens, 50021 columns 567, 411, 382 (three rounds and the rest 327).
// 128 x 128 and 128 x 64 tiles were within 3 % of the best of the three at
// most, and are not built.
struct CeTile {
  int mt, nt, slots;  // slots: workgroups a CU
  double lo, hi, tbs;
};
constexpr CeTile kCeTiles[3] = {{1, 2, 2, 0.21, 0.74, 6.9}, {2, 4, 1, 0.98, 0.99, 6.8},
                                {4, 4, 1, 1.23, 1.51, 5.3}};

static int64_t ceil_to(int64_t a, int64_t b) { return (a + b - 1) / b; }

static double ce_cost(const CeTile &c, int64_t m, int64_t v, int64_t d) {
  const int64_t tl = ceil_to(m, 64 * c.mt), T = tl * ceil_to(v, 64 * c.nt);
  const int64_t slots = (int64_t)cu_slots() * c.slots;
  const double steps = (double)ceil_to(d, kGcStep);
  const double part = (double)(T % slots) / (double)slots;
  const double compute =
      steps * ((double)(T / slots) * c.hi + (part > 0.0 ? c.lo + (c.hi - c.lo) * part : 0.0));
  const double memory = 2e-6 * (double)v * (double)d / c.tbs * (0.79 + 0.21 * (double)tl);
  return 8.0 + (compute > memory ? compute : memory);
}

static int ce_tiles(int64_t m, int64_t v, int64_t d, CeLaunch (&out)[2]) {
  double best = HUGE_VAL;
  int count = 0;
  auto smallest = [&](int64_t cols, int upto, const CeTile *&c) {
    double least = HUGE_VAL;
    for (int i = 0; i < upto; ++i) {
      const double t = ce_cost(kCeTiles[i], m, cols, d);
      if (t < least) {
        least = t;
        c = &kCeTiles[i];
      }
    }
    return least;
  };
  const CeTile *c = nullptr;
  best = smallest(v, 3, c);
  out[0] = CeLaunch{c->mt, c->nt, v};
  count = 1;
  for (int i = 1; i < 3; ++i) {
    const CeTile &a = kCeTiles[i];
    const int64_t tl = ceil_to(m, 64 * a.mt), T = tl * ceil_to(v, 64 * a.nt);
    const int64_t rounds = T / cu_slots();
    const int64_t cols = rounds * cu_slots() / tl * (64 * a.nt);
    if (rounds == 0 || cols == 0 || cols >= v) continue;
    const double t = ce_cost(a, m, cols, d) + smallest(v - cols, i, c);
    if (t < best) {
      best = t;
      out[0] = CeLaunch{a.mt, a.nt, cols};
      out[1] = CeLaunch{c->mt, c->nt, v - cols};
      count = 2;
    }
  }
  return count;
}

// Partial sums a token leaves: one for each half tile.
static int64_t ce_slices(int64_t m, int64_t v, int64_t d) {
  CeLaunch l[2];
  const int n = ce_tiles(m, v, d, l);
  int64_t s = 0;
  for (int i = 0; i < n; ++i) s += 2 * ceil_to(l[i].cols, 64 * l[i].nt);
  return s;
}

struct CePlan {
  int64_t tokens;        // forward: tokens of one launch
  int64_t part_bytes, fwd_bytes;
  int64_t piece, ldg;    // backward: columns of a piece, row length of G
  int dx_mt;
  int64_t slices, slice; // of dx's reduction over a piece
  int64_t g_bytes, bwd_bytes;
};

// Tile height of dx and slices of its reduction over a piece, by the least of:
// the rounds' time, as for the logits, joined with that of reading w by their
// fourth powers (the larger one, a little more where they are close); what the
// slices' fp32 sums move at 2.4 TB/s (written, read and written by each further
// piece, read for the join).  Fitted to 1 to 4096 tokens, 8000 to 50021
// columns, d = 1024 to 8192, all heights and 1 to 32 slices; measured again with
// the present products at 72 shapes of 1 to 4096 tokens, 8000 to 128000 columns:
// 0.1 % from the best on average, 3 % at most.  The gradients of 777 x 32000 x
// 4096: 615 us with tiles of 128 rows x 2 slices, 616 with 256 rows x 4, 938 and
// 999 with 64 and 256 rows in one.
constexpr CeTile kCeDxTiles[3] = {{1, 4, 2, 0.75, 0.97, 5.0}, {2, 4, 1, 0.61, 0.88, 5.0},
                                  {4, 4, 1, 0.95, 1.03, 5.0}};
static void ce_dx_plan(int64_t m, int64_t v, int64_t d, CePlan &p) {
  const double pieces = (double)ceil_to(v, p.piece);
  const int64_t steps = ceil_to(p.ldg, kGcStep);
  double best = HUGE_VAL;
  for (const CeTile &c : kCeDxTiles) {
    const int64_t tl = ceil_to(m, 64 * c.mt), T = tl * ceil_to(d, 64 * c.nt);
    const int64_t slots = (int64_t)cu_slots() * c.slots;
    for (int64_t s = 1; s <= 32 && (s == 1 || steps >= 4 * s) && T * s <= kMaxTiles; ++s) {
      const int64_t each = ceil_to(steps, s), n = T * ceil_to(steps, each);
      const double part = (double)(n % slots) / (double)slots;
      const double compute =
          (double)each *
          ((double)(n / slots) * c.hi + (part > 0.0 ? c.lo + (c.hi - c.lo) * part : 0.0));
      const double memory =
          2e-6 * (double)p.piece * (double)d / c.tbs * (0.75 + 0.25 * (double)tl);
      const double sums = 8e-6 * (double)(n / T) * (double)m * (double)d / 2.4;
      const double c2 = compute * compute, m2 = memory * memory;
      const double cost = pieces * (sums + std::sqrt(std::sqrt(c2 * c2 + m2 * m2)));
      if (cost < best) {
        best = cost;
        p.dx_mt = c.mt;
        p.slice = each * kGcStep;
      }
    }
  }
  p.slices = ceil_to(p.ldg, p.slice);
}

static int32_t ce_plan(int64_t m, int64_t v, int64_t d, CePlan &p) {
  if (m < 0 || v <= 0 || d <= 0)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "bad cross-entropy shape m=%lld v=%lld d=%lld",
                (long long)m, (long long)v, (long long)d);
  if (d % 8 != 0)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "cross entropy needs d %% 8 == 0, got %lld",
                (long long)d);
  // Offsets within a tile's step and tile counts are 32-bit.
  if (d > ((int64_t)1 << 20) || v > ((int64_t)1 << 28) || m > ((int64_t)1 << 24))
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE,
                "cross entropy of m=%lld v=%lld d=%lld beyond m 2^24, v 2^28, d 2^20",
                (long long)m, (long long)v, (long long)d);
  p.tokens = m < kCeTokens ? m : kCeTokens;
  p.part_bytes = m > 0 ? ce_slices(p.tokens, v, d) * p.tokens : 0;
  if (m > 0 && m % p.tokens != 0) {
    const int64_t last = ce_slices(m % p.tokens, v, d) * (m % p.tokens);
    if (last > p.part_bytes) p.part_bytes = last;
  }
  p.part_bytes = up(p.part_bytes * 8, 256);
  p.fwd_bytes = p.part_bytes + p.tokens * 4;
  int64_t most = m > 0 ? kCePieceBytes / (2 * m) / 256 * 256 : v;
  most = most < 256 ? 256 : (most > (1 << 20) ? (1 << 20) : most);
  const int64_t pieces = (v + most - 1) / most;
  p.piece = up((v + pieces - 1) / pieces, 256);
  if (p.piece > v) p.piece = v;
  p.ldg = up(p.piece, 64);
  // Tiles of the forward, of a piece's logits and dw, and of dx, at the smallest
  // tiles of each.
  if (ceil_to(p.tokens, 64) * ceil_to(v, 128) > kMaxTiles ||
      ceil_to(m, 64) * ceil_to(p.piece, 128) > kMaxTiles ||
      ceil_to(p.piece, 128) * ceil_to(d, 128) > kMaxTiles ||
      ceil_to(m, 64) * ceil_to(d, 256) > kMaxTiles)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "too many tiles");
  ce_dx_plan(m, v, d, p);
  p.g_bytes = up(m * p.ldg * 2, 256);
  p.bwd_bytes = p.g_bytes + p.slices * m * d * 4 + 16;  // G, dx's sums, c
  return NF4S_OK;
}

// The logits of a.M tokens and a.vn columns, in one launch or two; *slices: the
// partial sums of a token.
template <bool kGrad>
static int32_t ce_logits(CeLogits a, int64_t *slices, hipStream_t s) {
  CeLaunch l[2];
  const int n = ce_tiles(a.M, a.vn, a.d, l);
  int64_t done = 0;
  for (int i = 0; i < n; ++i) {
    a.vn = (int32_t)l[i].cols;
    a.tiles_l = (int32_t)ceil_to(a.M, 64 * l[i].mt);
    a.tiles_r = (int32_t)ceil_to(a.vn, 64 * l[i].nt);
    a.strip = kCeStrip;
    auto *kernel = l[i].mt == 4   ? ce_logits_kernel<4, 4, kGrad>
                   : l[i].mt == 2 ? ce_logits_kernel<2, 4, kGrad>
                                  : ce_logits_kernel<1, 2, kGrad>;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)a.tiles_l * (uint32_t)a.tiles_r), dim3(kGcThreads),
                       0, s, a);
    const int32_t rc = check_launch("ce_logits_kernel");
    if (rc != NF4S_OK) return rc;
    a.w += a.vn * a.d;
    a.v0 += a.vn;
    if (kGrad) a.g += a.vn;
    if (!kGrad) a.part += 2 * a.tiles_r * a.M;
    a.gcols -= a.vn;
    done += 2 * a.tiles_r;
  }
  if (slices != nullptr) *slices = done;
  return NF4S_OK;
}

template <int kMT, int kNT, bool kLAcross, int kOut>
static int32_t ce_product(CeProduct a, hipStream_t s) {
  a.tiles_l = (int32_t)ceil_to(a.rows, 64 * kMT);
  a.tiles_r = (int32_t)ceil_to(a.cols, 64 * kNT);
  a.strip = kCeStrip;
  const int64_t slices = (a.k + a.slice - 1) / a.slice;
  auto *kernel = ce_product_kernel<kMT, kNT, kLAcross, kOut>;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)(slices * a.tiles_l * a.tiles_r)), dim3(kGcThreads), 0,
                     s, a);
  return check_launch("ce_product_kernel");
}

template <int kOut>
static int32_t ce_dx_piece(const CePlan &p, const CeProduct &a, hipStream_t s) {
  return p.dx_mt == 4   ? ce_product<4, 4, false, kOut>(a, s)
         : p.dx_mt == 2 ? ce_product<2, 4, false, kOut>(a, s)
                        : ce_product<1, 4, false, kOut>(a, s);
}

template <int kOut>
static int32_t ce_dw_piece(const CeProduct &a, hipStream_t s) {
  return a.k <= kCeFewTokens ? ce_product<2, 2, true, kOut>(a, s)
                             : ce_product<4, 4, true, kOut>(a, s);
}

static int32_t ce_operands(const uint16_t *x, const uint16_t *w, const int64_t *targets, int64_t m,
                           void *workspace, int64_t workspace_bytes, int64_t need) {
  if (w == nullptr || (m > 0 && (x == nullptr || targets == nullptr)))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
  if (!aligned(w, 16) || (m > 0 && (!aligned(x, 16) || !aligned(targets, 8))))
    return fail(NF4S_ERR_MISALIGNED, "x and w must be 16-byte aligned, targets 8-byte");
  if (m > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "cross entropy needs %lld workspace bytes",
                (long long)need);
  if (m > 0 && !aligned(workspace, 16))
    return fail(NF4S_ERR_MISALIGNED, "workspace must be 16-byte aligned");
  return NF4S_OK;
}

}  // namespace nf4s

using namespace nf4s;

extern "C" {

int32_t nf4s_linear_ce_workspace_size(int64_t m, int64_t v, int64_t d, int32_t backward,
                                      int64_t *bytes) {
  clear_error();
  if (bytes == nullptr) return fail(NF4S_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = 0;
  CePlan p;
  const int32_t rc = ce_plan(m, v, d, p);
  if (rc == NF4S_OK && m > 0) *bytes = backward ? p.bwd_bytes : p.fwd_bytes;
  return rc;
}

int32_t nf4s_linear_ce_fwd(const uint16_t *x, const uint16_t *w, const int64_t *targets, int64_t m,
                           int64_t v, int64_t d, int64_t ignore_index, float *loss, float *lse,
                           void *workspace, int64_t workspace_bytes, void *stream) {
  clear_error();
  CePlan p;
  int32_t rc = ce_plan(m, v, d, p);
  if (rc != NF4S_OK || m == 0) return rc;
  rc = ce_operands(x, w, targets, m, workspace, workspace_bytes, p.fwd_bytes);
  if (rc != NF4S_OK) return rc;
  if (loss == nullptr || lse == nullptr)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "loss or lse is NULL");
  if (!aligned(loss, 4) || !aligned(lse, 4))
    return fail(NF4S_ERR_MISALIGNED, "loss and lse must be 4-byte aligned");
  const hipStream_t s = as_stream(stream);
  CeLogits a{};
  a.w = w;
  a.d = d;
  a.vn = (int32_t)v;
  a.V = v;
  a.ignore = ignore_index;
  a.part = static_cast<floatx2 *>(workspace);
  a.zt = reinterpret_cast<float *>(static_cast<char *>(workspace) + p.part_bytes);
  for (int64_t m0 = 0; m0 < m; m0 += p.tokens) {
    a.M = m - m0 < p.tokens ? m - m0 : p.tokens;
    a.x = x + m0 * d;
    a.targets = targets + m0;
    int64_t slices = 0;
    rc = ce_logits<false>(a, &slices, s);
    if (rc != NF4S_OK) return rc;
    const bool few = a.M < 512;
    hipLaunchKernelGGL(few ? ce_join_kernel<1> : ce_join_kernel<8>,
                       dim3((uint32_t)(few ? a.M : (a.M + 7) / 8)), dim3(256), 0, s, a.part, a.zt,
                       a.targets, a.M, (int32_t)slices, v, ignore_index, loss + m0, lse + m0);
    rc = check_launch("ce_join_kernel");
    if (rc != NF4S_OK) return rc;
  }
  return NF4S_OK;
}

int32_t nf4s_linear_ce_bwd(const uint16_t *x, const uint16_t *w, const int64_t *targets,
                           const float *lse, const float *dloss, int64_t m, int64_t v, int64_t d,
                           int64_t ignore_index, uint16_t *dx, void *dw, int32_t dw_is_f32,
                           int32_t accumulate, void *workspace, int64_t workspace_bytes,
                           void *stream) {
  clear_error();
  CePlan p;
  int32_t rc = ce_plan(m, v, d, p);
  if (rc != NF4S_OK) return rc;
  rc = ce_operands(x, w, targets, m, workspace, workspace_bytes, p.bwd_bytes);
  if (rc != NF4S_OK) return rc;
  if (accumulate && !dw_is_f32)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "dw accumulates in fp32 only");
  if (dw == nullptr || (m > 0 && (lse == nullptr || dloss == nullptr || dx == nullptr)))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "lse, dloss, dx or dw is NULL");
  if (!aligned(dw, 16) || (m > 0 && (!aligned(dx, 16) || !aligned(lse, 4) || !aligned(dloss, 4))))
    return fail(NF4S_ERR_MISALIGNED, "dx and dw must be 16-byte aligned, lse and dloss 4-byte");
  const hipStream_t s = as_stream(stream);
  if (m == 0) {
    if (accumulate) return NF4S_OK;
    const int64_t n = dw_is_f32 ? v * d : v * d / 2;  // 32-bit words
    hipLaunchKernelGGL(ce_zero_kernel<uint32_t>, dim3(4096), dim3(256), 0, s,
                       static_cast<uint32_t *>(dw), n);
    return check_launch("ce_zero_kernel");
  }
  uint16_t *g = static_cast<uint16_t *>(workspace);
  float *part = reinterpret_cast<float *>(static_cast<char *>(workspace) + p.g_bytes);
  float *common = part + p.slices * m * d;
  hipLaunchKernelGGL(ce_common_kernel, dim3(1), dim3(1024), 0, s, dloss, targets, ignore_index, m,
                     common);
  rc = check_launch("ce_common_kernel");
  if (rc != NF4S_OK) return rc;
  for (int64_t v0 = 0; v0 < v; v0 += p.piece) {
    const int64_t vn = v - v0 < p.piece ? v - v0 : p.piece;
    CeLogits a{};
    a.x = x;
    a.w = w + v0 * d;
    a.targets = targets;
    a.M = m;
    a.d = d;
    a.v0 = v0;
    a.vn = (int32_t)vn;
    a.V = v;
    a.ignore = ignore_index;
    a.lse = lse;
    a.dloss = dloss;
    a.common = common;
    a.g = g;
    a.ldg = a.gcols = p.ldg;
    rc = ce_logits<true>(a, nullptr, s);
    if (rc != NF4S_OK) return rc;
    CeProduct b{};  // dx += G . w
    b.l = g;
    b.ldl = p.ldg;
    b.r = w + v0 * d;
    b.ldr = d;
    b.rows = m;
    b.cols = d;
    b.k = vn;
    b.slice = p.slice;
    b.out = part;
    b.ld = d;
    b.slice_stride = m * d;
    rc = v0 == 0 ? ce_dx_piece<kOutF32>(p, b, s) : ce_dx_piece<kOutF32Add>(p, b, s);
    if (rc != NF4S_OK) return rc;
    CeProduct c{};  // the piece's rows of dw = G^T . x
    c.l = g;
    c.ldl = p.ldg;
    c.r = x;
    c.ldr = d;
    c.rows = vn;
    c.cols = d;
    c.k = m;
    c.slice = up(m, kGcStep);
    c.out = dw_is_f32 ? static_cast<void *>(static_cast<float *>(dw) + v0 * d)
                      : static_cast<void *>(static_cast<uint16_t *>(dw) + v0 * d);
    c.ld = d;
    c.common = common;
    rc = accumulate  ? ce_dw_piece<kOutF32Add>(c, s)
         : dw_is_f32 ? ce_dw_piece<kOutF32>(c, s)
                     : ce_dw_piece<kOutBf16>(c, s);
    if (rc != NF4S_OK) return rc;
  }
  const int64_t chunks = m * d / 4;
  const int64_t blocks = (chunks + 255) / 256;
  hipLaunchKernelGGL(ce_dx_kernel, dim3((uint32_t)(blocks < 65536 ? blocks : 65536)), dim3(256), 0,
                     s, reinterpret_cast<const floatx4 *>(part), (int32_t)p.slices, chunks,
                     common, reinterpret_cast<u32x2 *>(dx));
  return check_launch("ce_dx_kernel");
}

}  // extern "C"
