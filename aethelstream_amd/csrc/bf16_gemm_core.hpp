// bf16_gemm_core.hpp - the tile product of the loss head's three bf16 GEMMs on
// gfx950 (MI355X): out[l, r] = sum_k L[l, k] R[r, k], each operand stored
// either along the reduction (rows of k) or across it (rows of l or r).
//
//   logits  X . W^T   both along
//   dX      P . W     L along, R across
//   dW      P^T . X   both across
//
// Workgroup = 4 waves in 2 x 2, tile = 64 kMT rows (l) x 64 kNT columns (r);
// each wave owns 32 kMT x 32 kNT in 2 kMT x 2 kNT accumulators of
// v_mfma_f32_16x16x32_bf16, R as the instruction's first operand: a lane holds
// one row l of each accumulator and four adjacent columns.  (These products are
// bound by power, and 32x32x16 takes more: from registers alone random operands
// sustain 2.05 PFLOP/s with 16x16x32 and 1.81 with 32x32x16, with the LDS reads
// of 128 x 128 a wave 1.71 and 1.63.)
// Per 64-long step both operands' tiles move into LDS with direct-to-LDS loads,
// into rings of kNL and kNR stages: while step t computes, L of step t + kNL - 1
// and R of step t + kNR - 1 are on their way.  An operand along the reduction is
// read with ds_read_b128, 8 consecutive k of one row a lane; one across it with
// the transposing ds_read_b64_tr_b16.
#pragma once

#include "abi_common.hpp"
#include "gemm_common.hpp"
#include "nf4_device.hpp"
#include "tr_tile.hpp"

namespace nf4s {

constexpr int kGcThreads = 256;
constexpr int kGcStep = 64;

// One operand of a tile product, `ld` elements a row, from `p`: the tile's first
// row (along), or the first k row at the tile's first column (across).  `left`
// bytes from p may be read, a multiple of 16 from each row's start; what lies
// past them reads as zero.
struct GcOperand {
  const uint16_t *p;
  int64_t ld, left;
};
// Along: `rows` rows of k elements (a multiple of 8).  Across: k rows, `cols`
// elements of each from p on.
__device__ __forceinline__ GcOperand gc_along(const uint16_t *p, int64_t ld, int64_t rows,
                                              int64_t k) {
  return GcOperand{p, ld, rows > 0 ? ((rows - 1) * ld + k) * 2 : 0};
}
__device__ __forceinline__ GcOperand gc_across(const uint16_t *p, int64_t ld, int64_t cols,
                                               int64_t k) {
  return GcOperand{p, ld, k > 0 ? ((k - 1) * ld + cols) * 2 : 0};
}

// LDS tile of an operand along the reduction: rows of 128 bytes, 8 units of 16.
// Unit u of row r lives at physical unit u ^ gc_swz(r).  With r & 7 the fragment
// reads (16 rows of 4 units a wave) have no bank conflicts.  Tiles of 256 x 256
// have a second term, which doubles half the banks' accesses and is faster there
// nonetheless: 4096 x 32000 x 8192 forward 1520 us and 1521 without, the median of
// five 1536 and 1559, gradients 4641 and 4693.  In smaller tiles it makes no
// difference while w comes from memory (77 x 32000 x 4096 67 us either way), 2 to 4
// % where it is in the caches.  (Times of this file: whole calls, the variants in
// turn on one card, the least of five.)
template <bool kWide>
__device__ __forceinline__ int gc_swz(int row) {
  return (row & 7) ^ (kWide ? (row >> 3) & 1 : 0);
}

// LDS tile of an operand across it: k rows of kUnits (32 or 16) units.  Unit u
// of row r lives at physical unit (u & 16) | ((u & 15) ^ s(r)): each 32-lane half
// of a transposed fragment read, 8 rows of 2 units each, covers 16 distinct units
// of one half-row's 64 banks, and each 16-lane quarter of a DMA writes one row's
// 16 contiguous units.
__device__ __forceinline__ int gc_unit(int row, int u) {
  return (u & 16) | ((u & 15) ^ (5 * (row & 3)) ^ (2 * ((row >> 3) & 1)));
}

template <int kTiles, bool kAcross, bool kWide>
struct GcSide {
  static constexpr int kBytes = 8192 * kTiles;   // of one stage
  static constexpr int kUnits = 8 * kTiles;      // across: units of a k row
  static constexpr int kDmas = 2 * kTiles;       // per wave and step
  static constexpr int kFrags = 2 * kTiles;      // of 16 rows, per wave and sub-step
  static constexpr int kAddrs = kAcross ? 1 : 2;
  static_assert(!kAcross || kUnits >= 16, "gc_unit");

  // Lane addresses of the fragment reads: lane l reads row (along) or column
  // (across) l % 16 of its fragment, k = 8 (l / 16) + 0..7 of the sub-step of 32.
  // Across (transposing reads): lane 4e + c of a 16-lane group addresses k row e,
  // columns 4c..4c+3, and receives the four rows of column l % 16; a second read
  // 4 rows lower completes the 8.  Fragment j, 2 units further on, is 32 j away in
  // bits 5 to 7, which nothing but the unit sets (a row is a multiple of 256
  // bytes, a stage of 8192).  Along one address per sub-step, fragments are 16
  // rows = 2048 bytes apart.
  static __device__ __forceinline__ void read_addrs(uint32_t (&a)[kAddrs], int lane, int half) {
    if constexpr (kAcross) {
      const int l16 = lane & 15;
      const int row = 8 * (lane >> 4) + (l16 >> 2);
      const int u = kUnits / 2 * half + ((l16 >> 1) & 1);
      a[0] = (uint32_t)(16 * (kUnits * row + gc_unit(row, u)) + 8 * (l16 & 1));
    } else {
      const int row = 32 * kTiles * half + (lane & 15);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        a[s] = (uint32_t)(128 * row + 16 * ((4 * s + (lane >> 4)) ^ gc_swz<kWide>(row)));
    }
  }
  static __device__ __forceinline__ u32x4 frag(const char *base, const uint32_t (&a)[kAddrs],
                                               int s, int j) {
    if constexpr (kAcross)
      return tr_frag<kUnits>(base, (a[0] ^ (32 * j)) + 512 * kUnits * s);
    else
      return *reinterpret_cast<const u32x4 *>(base + a[s] + 2048 * j);
  }

  // Byte offsets of this wave's DMAs from the operand's place at a step.
  static __device__ __forceinline__ void dma_offsets(uint32_t (&v)[kDmas], int64_t ld, int lane,
                                                     int wave) {
#pragma unroll
    for (int q = 0; q < kDmas; ++q) {
      if constexpr (kAcross) {
        constexpr int kRows = 64 / kUnits;  // k rows per instruction
        const int r = 16 * wave + kRows * q + lane / kUnits;
        v[q] = (uint32_t)(r * ld * 2 + 16 * gc_unit(r, lane % kUnits));
      } else {
        const int r = 8 * (kDmas * wave + q) + (lane >> 3);
        v[q] = (uint32_t)(r * ld * 2 + 16 * ((lane & 7) ^ gc_swz<kWide>(r)));
      }
    }
  }
  // Along, last step of a reduction that ends inside it: units past the end are
  // moved out of range, where loads give zero.
  static __device__ __forceinline__ void mask_tail(uint32_t (&v)[kDmas], int tail, int lane,
                                                   int wave) {
    if constexpr (!kAcross) {
#pragma unroll
      for (int q = 0; q < kDmas; ++q) {
        const int r = 8 * (kDmas * wave + q) + (lane >> 3);
        if (8 * ((lane & 7) ^ gc_swz<kWide>(r)) >= tail) v[q] = 0x80000000u;
      }
    }
  }
  // LDS offset of this wave's DMA q.
  static __device__ __forceinline__ int dma_lds(int q, int wave) {
    return 1024 * (kDmas * wave + q);
  }
};

// The place of an operand at a step: base pointer and bytes from it to the end
// of what may be read.
struct GcPlace {
  const char *p;
  int64_t left;
  int64_t step;  // bytes from one step to the next
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    const int64_t n = left < 0 ? 0 : (left > 0x7fffffff ? 0x7fffffff : left);
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)n, kBufferFlags);
  }
  __device__ __forceinline__ void advance() {
    p += step;
    left -= step;
  }
};

// Stages of the rings.  256 x 256 tiles: 3 of L and 2 of R are the 160 KB of a
// CU.  64 x 256 and 128 x 128 tiles: 2 of each, and two workgroups a CU; 64 x
// 128: 3 of each and two workgroups; 64 x 64: 5 of each and two workgroups, also the
// 160 KB.
template <int kMT, int kNT>
constexpr int kGcStagesL = kMT * kNT == 4 ? 2 : kMT * kNT == 1 ? 5 : 3;
template <int kMT, int kNT>
constexpr int kGcStagesR = kMT * kNT == 4 || kMT * kNT == 16 ? 2 : kMT * kNT == 1 ? 5 : 3;

template <int kMT, int kNT, bool kLAcross, bool kRAcross>
struct GcCore {
  static constexpr bool kWide = kMT * kNT == 16;
  using LSide = GcSide<kMT, kLAcross, kWide>;
  using RSide = GcSide<kNT, kRAcross, kWide>;
  static constexpr int kTileL = 64 * kMT, kTileR = 64 * kNT;
  static constexpr int kNL = kGcStagesL<kMT, kNT>, kNR = kGcStagesR<kMT, kNT>;
  static_assert(kNL == kNR || (kNL == 3 && kNR == 2), "kInFlight below");
  static constexpr int kPeriod = kNL == kNR ? kNL : 6;  // steps until both rings are back
  // DMAs that may be in flight when step t closes, those of steps t + 2 to t + kNL - 1:
  // all, or of step t + 2 L's.
  static constexpr int kInFlight =
      kNL == kNR ? (kNL - 2) * (LSide::kDmas + RSide::kDmas) : LSide::kDmas;
  static constexpr int kLdsBytes = kNL * LSide::kBytes + kNR * RSide::kBytes;
  static constexpr int kFL = LSide::kFrags, kFR = RSide::kFrags;
  static constexpr int kSub = kFL * kFR;       // MFMAs per sub-step of 32
  static constexpr int kPost = 3 * kSub / 8;   // those that open the next step
  static constexpr int kFront = 2 * kSub - kPost;
  static constexpr int kReads = kFL + kFR;
  // From 128 accumulator registers on, the instruction is written out with the
  // sum's registers as its own source.  Left to the compiler the sums move: from
  // 50 to 200 copies a step of 128 MFMAs, and 4096 x 32000 x 8192 logits take 1946 us
  // (1520 tied).  The compiler does not know that the block is an MFMA, so the
  // waits that it would add are this file's: the fragments come from LDS reads,
  // which it waits for, never from an instruction of the two before; the sums
  // stay where they are until run() has waited for the last of them.
  // (Checked in the listing by test_loss_listing.py.)
  static constexpr bool kTied = kSub >= 32;
  static constexpr int kDmas = LSide::kDmas + RSide::kDmas;
  // MFMAs from one DMA to the next: spread over what follows the opening, as the
  // reads and the DMAs together keep LDS busy for three quarters of a 256 x 256
  // step at the MFMA rate.  4096 x 32000 x 8192 logits: 1520 us; with half a
  // sub-step in the opening, a gap of 5 1526 and of 4 1568.
  static constexpr int kGap = (kFront - 1) / kDmas;
  static_assert(kDmas <= kFront, "one DMA per MFMA slot at most");

  floatx4 acc[kFL][kFR];
  u32x4 fl[2][kFL], fr[2][kFR];
  uint32_t al[LSide::kAddrs], ar[RSide::kAddrs];
  uint32_t vl[LSide::kDmas], vr[RSide::kDmas];
  GcPlace pl, pr;

  // Fragment read q of a sub-step, in the order its MFMAs use them: l0, r0, r1,
  // .., l1, ..
  __device__ __forceinline__ void read(const char *lds, int s, int b, int q) {
    if (q == 0 || q > kFR) {
      const int j = q == 0 ? 0 : q - kFR;
      fl[b][j] = LSide::frag(lds, al, s, j);
    } else {
      fr[b][q - 1] = RSide::frag(lds, ar, s, q - 1);
    }
  }
  template <int kI>
  __device__ __forceinline__ void mfma(int b) {
    constexpr int mt = kI / kFR, nt = kI % kFR;
    if constexpr (kTied)
      asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0"
                   : "+a"(acc[mt][nt])
                   : "v"(fr[b][nt]), "v"(fl[b][mt]));
    else
      acc[mt][nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
          __builtin_bit_cast(bf16x8, fr[b][nt]), __builtin_bit_cast(bf16x8, fl[b][mt]), acc[mt][nt],
          0, 0, 0);
  }
  // DMA d of a step: R's, which are needed first, then L's.
  template <int kD>
  __device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t rl, __amdgpu_buffer_rsrc_t rr,
                                      char *nl, char *nr, bool more_l, bool more_r, int wave) {
    if constexpr (kD < RSide::kDmas) {
      if (more_r)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rr, (lds_void_t *)(nr + RSide::dma_lds(kD, wave)), 16, (int)vr[kD], 0, 0, 0);
    } else {
      constexpr int d = kD - RSide::kDmas;
      if (more_l)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rl, (lds_void_t *)(nl + LSide::dma_lds(d, wave)), 16, (int)vl[d], 0, 0, 0);
    }
  }

  // One step from the stages that al and ar address: the previous step's last
  // kPost MFMAs with the reads of sub-step 0 between them, then 2 sub-steps of
  // kSub, the fragments of sub-step 1 read during sub-step 0, the DMAs of the
  // steps ahead (if they exist) into stages `nl`/`nr` between the MFMAs.  Those
  // stages were last read in step t - 1, whose reads ended before the barrier
  // that closed it.  The __restrict__ stages tell the compiler that DMAs into
  // one never alias reads of the other, so that it waits for them at the
  // barriers only.
  __device__ __forceinline__ void step(const char *__restrict__ lds, char *__restrict__ nl,
                                       char *__restrict__ nr, bool more_l, bool more_r, int wave) {
    const __amdgpu_buffer_rsrc_t rl = pl.rsrc(), rr = pr.rsrc();
    static_for<0, kPost>([&](auto I) {
      constexpr int i = decltype(I)::value;
      mfma<kSub - kPost + i>(1);
      static_for<0, kReads>([&](auto Q) {
        constexpr int q = decltype(Q)::value;
        if constexpr (q * kPost / kReads == i) read(lds, 0, 0, q);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    static_for<0, kFront>([&](auto N) {
      constexpr int n = decltype(N)::value;
      constexpr int s = n / kSub, i = n % kSub;
      mfma<i>(s & 1);
      if constexpr (s == 0) {
        static_for<0, kReads>([&](auto Q) {
          constexpr int q = decltype(Q)::value;
          if constexpr (q * kSub / kReads == i) read(lds, 1, 1, q);
        });
      }
      if constexpr (n % kGap == 0 && n / kGap < kDmas) {
        dma<n / kGap>(rl, rr, nl, nr, more_l, more_r, wave);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  // Read addresses from stage kI % kN of a ring to the next.  Opaque, as the
  // compiler would keep the addresses of every stage in registers.
  template <int kBytes, int kN, int kI, int kA>
  static __device__ __forceinline__ void move(uint32_t (&a)[kA]) {
#pragma unroll
    for (int i = 0; i < kA; ++i) {
      a[i] += (kI % kN == kN - 1 ? 1 - kN : 1) * kBytes;
      asm volatile("" : "+v"(a[i]));
    }
  }

  // The barrier that closes step t: this wave's DMAs of step t + 1 have landed
  // and its LDS reads of step t have ended.  Those of the steps from t + 2 on that are
  // already issued may be in flight: they were issued after step t + 1's.  (Where the
  // last of them is missing, none may.)
  static __device__ __forceinline__ void close_step(int t, int nsteps) {
    if (t + (kNL > 3 ? kNL - 1 : 2) < nsteps)
      step_barrier<kInFlight>();
    else
      step_barrier<0>();
  }

  // The whole product into acc: k elements of the reduction, lds of kLdsBytes.
  // With k no multiple of 8, an operand along the reduction holds zeros (and may
  // be read) up to the next one.
  __device__ __forceinline__ void run(const GcOperand &l, const GcOperand &r, int64_t k, char *lds,
                                      int lane, int wave) {
    char *sl[kNL], *sr[kNR];
#pragma unroll
    for (int i = 0; i < kNL; ++i) sl[i] = lds + i * LSide::kBytes;
#pragma unroll
    for (int i = 0; i < kNR; ++i) sr[i] = lds + kNL * LSide::kBytes + i * RSide::kBytes;
    LSide::read_addrs(al, lane, wave >> 1);
    RSide::read_addrs(ar, lane, wave & 1);
#pragma unroll
    for (int i = 0; i < RSide::kAddrs; ++i) ar[i] += kNL * LSide::kBytes;
    LSide::dma_offsets(vl, l.ld, lane, wave);
    RSide::dma_offsets(vr, r.ld, lane, wave);
    pl = place<kLAcross>(l);
    pr = place<kRAcross>(r);
    const int nsteps = (int)((k + kGcStep - 1) / kGcStep);
    const int tail = (int)(k % kGcStep);
    // Called with the step whose DMAs are next.
    auto mask_l = [&](int t) {
      if (tail != 0 && t == nsteps - 1) LSide::mask_tail(vl, tail, lane, wave);
    };
    auto mask_r = [&](int t) {
      if (tail != 0 && t == nsteps - 1) RSide::mask_tail(vr, tail, lane, wave);
    };
    static_for<0, kNL - 1>([&](auto P) {
      constexpr int t = decltype(P)::value;
      mask_l(t);
      mask_r(t);
      const __amdgpu_buffer_rsrc_t rl = pl.rsrc(), rr = pr.rsrc();
      static_for<t < kNR - 1 ? 0 : RSide::kDmas, kDmas>([&](auto D) {
        dma<decltype(D)::value>(rl, rr, sl[t], sr[t % kNR], t < nsteps, t < nsteps, wave);
      });
      pl.advance();
      if (t < kNR - 1) pr.advance();
    });
#pragma unroll
    for (int mt = 0; mt < kFL; ++mt)
#pragma unroll
      for (int nt = 0; nt < kFR; ++nt) acc[mt][nt] = (floatx4){0.0f, 0.0f, 0.0f, 0.0f};
    // The first step's opening MFMAs multiply zeros.
#pragma unroll
    for (int i = 0; i < kFL; ++i) fl[1][i] = (u32x4){0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kFR; ++i) fr[1][i] = (u32x4){0u, 0u, 0u, 0u};
    close_step(-1, nsteps);
    int t = 0;
    auto one = [&](auto P) {
      constexpr int i = decltype(P)::value;
      mask_l(t + kNL - 1);
      mask_r(t + kNR - 1);
      step(lds, sl[(i + kNL - 1) % kNL], sr[(i + kNR - 1) % kNR], t + kNL - 1 < nsteps,
           t + kNR - 1 < nsteps, wave);
      pl.advance();
      pr.advance();
      move<LSide::kBytes, kNL, i>(al);
      move<RSide::kBytes, kNR, i>(ar);
      close_step(t, nsteps);
      ++t;
    };
#pragma unroll 1
    while (t + kPeriod <= nsteps) static_for<0, kPeriod>(one);
    static_for<0, kPeriod - 1>([&](auto P) {
      if (t < nsteps) one(P);
    });
    static_for<0, kPost>([&](auto I) { mfma<kSub - kPost + decltype(I)::value>(1); });
    if constexpr (kTied) {
      asm volatile("s_nop 15\n\ts_nop 3" ::: "memory");
#pragma unroll
      for (int mt = 0; mt < kFL; ++mt)
#pragma unroll
        for (int nt = 0; nt < kFR; ++nt) asm volatile("" : "+a"(acc[mt][nt]));
    }
  }

  template <bool kAcross>
  static __device__ __forceinline__ GcPlace place(const GcOperand &o) {
    return GcPlace{reinterpret_cast<const char *>(o.p), o.left,
                   kAcross ? kGcStep * o.ld * 2 : (int64_t)kGcStep * 2};
  }
};

// Tile b of a one-dimensional grid of tiles_l x tiles_r: numbered row by row
// within strips of `strip` tile columns, each XCD (workgroups b % 8) a
// contiguous range, so that an XCD's resident workgroups form a patch that
// shares its operands in that XCD's L2.
__device__ __forceinline__ void gc_tile(int b, int tiles_l, int tiles_r, int strip, int &tl,
                                        int &tr) {
  const int T = tiles_l * tiles_r;
  const int x = b & 7, base = T >> 3, rem = T & 7;
  const int n = x * base + (x < rem ? x : rem) + (b >> 3);
  const int per = tiles_l * strip;
  const int s = n / per, i = n - s * per;
  const int left = tiles_r - s * strip;
  const int w = left < strip ? left : strip;
  tl = i / w;
  tr = s * strip + i - tl * w;
}

// Orders a wave's own LDS writes before its reads of other lanes' values, and
// those reads before its next writes.
__device__ __forceinline__ void gc_wave_sync() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
  asm volatile("" ::: "memory");
}

// Stores 32 rows x 32 kNT columns of a wave as bf16 through its 32 * 64 * kNT
// bytes of LDS, whole rows of 64 kNT bytes: value(h, nt, i) is the lane's register
// i of row half h and column tile nt, already final.  `out` points at row 0, column 0 of the
// block; `rows` and `cols` (a multiple of 8) bound it.
template <int kNT, bool kNt, class F>
__device__ __forceinline__ void gc_store_bf16(F &&value, char *lds, uint16_t *out, int64_t ld,
                                              int64_t rows, int64_t cols, int lane) {
  constexpr int kChunks = 4 * kNT;  // 16-byte chunks of a row
  const int grp = lane >> 4;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int nt = 0; nt < 2 * kNT; ++nt) {
      const int row = 16 * h + (lane & 15);
      const u32x2 w = {pack_bf16x2(value(h, nt, 0), value(h, nt, 1)),
                       pack_bf16x2(value(h, nt, 2), value(h, nt, 3))};
      const int c = (2 * nt + (grp >> 1)) ^ (row & (kChunks - 1));
      *reinterpret_cast<u32x2 *>(lds + 16 * kChunks * row + 16 * c + 8 * (grp & 1)) = w;
    }
  gc_wave_sync();
  constexpr int kRows = 64 / kChunks;  // rows per store instruction
  const int r0 = lane / kChunks, c = lane % kChunks;
#pragma unroll
  for (int i = 0; i < 32 / kRows; ++i) {
    const int r = kRows * i + r0;
    const u32x4 w = *reinterpret_cast<const u32x4 *>(lds + 16 * kChunks * r +
                                                     16 * (c ^ (r & (kChunks - 1))));
    if (r < rows && 8 * c < cols) {
      u32x4 *p = reinterpret_cast<u32x4 *>(out + r * ld + 8 * c);
      if constexpr (kNt)
        __builtin_nontemporal_store(w, p);
      else
        *p = w;
    }
  }
  gc_wave_sync();
}

// The same for fp32 values, through 32 * 128 * kNT bytes; kAdd: added to what is
// there.
template <int kNT, bool kAdd, bool kNt, class F>
__device__ __forceinline__ void gc_store_f32(F &&value, char *lds, float *out, int64_t ld,
                                             int64_t rows, int64_t cols, int lane) {
  constexpr int kChunks = 8 * kNT;
  const int grp = lane >> 4;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int nt = 0; nt < 2 * kNT; ++nt) {
      const int row = 16 * h + (lane & 15);
      const int c = (4 * nt + grp) ^ (row & (kChunks - 1));
      *reinterpret_cast<floatx4 *>(lds + 16 * kChunks * row + 16 * c) =
          (floatx4){value(h, nt, 0), value(h, nt, 1), value(h, nt, 2), value(h, nt, 3)};
    }
  gc_wave_sync();
  constexpr int kRows = 64 / kChunks;
  const int r0 = lane / kChunks, c = lane % kChunks;
#pragma unroll
  for (int i = 0; i < 32 / kRows; ++i) {
    const int r = kRows * i + r0;
    floatx4 w = *reinterpret_cast<const floatx4 *>(lds + 16 * kChunks * r +
                                                   16 * (c ^ (r & (kChunks - 1))));
    if (r < rows && 4 * c < cols) {
      floatx4 *p = reinterpret_cast<floatx4 *>(out + r * ld + 4 * c);
      if constexpr (kAdd) w += *p;
      if constexpr (kNt)
        __builtin_nontemporal_store(w, p);
      else
        *p = w;
    }
  }
  gc_wave_sync();
}

}  // namespace nf4s
