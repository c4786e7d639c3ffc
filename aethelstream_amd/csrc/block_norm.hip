// block_norm.hip - the norms around a block with its gate and residual scale,
// forward and backward, for gfx950 (MI355X).
//
// Between two blocks of a decoder layer the reference adds the block's output to
// the residual and norms the sum for the next block (rms_norm_fwd,
// doublepass/src/math.rs:28-59, at doublepass/src/forward.rs:173 and :249).  Here
// that boundary is one kernel, with an optional norm of the block's output, an
// optional gate per channel and a residual scale:
//   h^ = h / rms(h),  u = w_post h^          (or h^ = u = h without w_post)
//   r' = r + alpha gate u                    (gate 1 without one)
//   y  = w_pre r' / rms(r'),  rms(v) = sqrt(mean(v^2) + eps)
// The forward reads h (bf16) and r (fp32) and writes r' (fp32) and y (bf16):
// 12 bytes an element.
//
// Backward, from dy (bf16) and the gradient dr' (fp32) that reached r' by the
// residual path.  With r^ = r' / rms_pre, e = w_pre dy, k = alpha gate w_post:
//   g  = dr' + (e - r^ mean(e r^)) / rms_pre         = dr
//   dh = (k g - h^ mean(k g h^)) / rms_post          (k g without w_post)
//   dw_pre = sum_rows dy r^,  S = sum_rows g h^,
//   dgate = alpha w_post S,   dw_post = alpha gate S.
// The gate and the norm's weight share one column sum, as both scale h^.  The
// second row mean needs g and so the first; it is taken from three sums of one
// pass, A = sum e r^, B = sum k h^ (dr' + e / rms_pre), C = sum k h^ r^:
//   sum k g h^ = B - (A / d) C / rms_pre,
// which costs one barrier a row instead of two.  18 bytes an element, 15.03
// where r' comes from its 8-bit checkpoint.  Both directions are bound by
// memory.
//
// A thread holds up to 4 (8) chunks of four elements, a workgroup of up to 1024
// threads a row, or several short ones.  Workgroups are persistent, with the
// next row on its way while one is worked on.  The backward's keep their column
// sums in registers, join those of their rows through LDS and write them once;
// a second kernel adds the workgroups' in order.
//
// Measured at 8192 x 8192: forward 132 us (6.1 TB/s; 154 with a workgroup a row,
// which reads the weights for every row), backward 215 to 221 us (5.5) and 4.6 for
// the columns; from a checkpoint at 4096 x 4096 52 us (4.8).  One row of 4096: 4
// us.  Whole calls there: without the block's norm and gate 134 and 213 us,
// without dres 181, without a block 165.
// Longer rows do not fit the registers: the forward past 16384 columns keeps 20 of
// a lane in scratch, the backward 52 (with a block) and 54, that of a block of
// 12292 to 16384 columns 8.  Whole calls of 4096 rows, forward and backward: 13824
// columns 121 and 271 us (5.6 and 3.8 TB/s), 16384 145 and 286 (5.6, 4.2), 28672
// 290 and 833 (4.9, 2.5), 32768 341 and 905 (4.7, 2.7; without a block 557).
#include "row_common.hpp"

namespace nf4s {

struct BlockNormFwd {
  const uint16_t *h;
  const float *res;
  const float *w_pre, *w_post, *gate;  // w_post, gate: NULL if absent
  float alpha, eps;
  int64_t m;
  int32_t chunks;  // d / 4
  float *res_out;  // may be res
  uint16_t *y;
  float *rms_pre, *rms_post;
};

// kKeep: rows of up to 4 chunks a thread; the weights stay in registers and the
// next row is on its way while this one is normed.  Longer rows read the weights
// again and load one row at a time.
template <int kMaxThreads, int kChunks, bool kKeep>
__global__ void __launch_bounds__(kMaxThreads) block_norm_fwd_kernel(const BlockNormFwd a) {
  __shared__ float part[2][16];
  const int threads = (int)blockDim.x;
  const bool post = a.w_post != nullptr;
  const float inv_d = 1.0f / (float)(4 * a.chunks);
  const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
  auto weight_k = [&](int c) {
    floatx4 k = {a.alpha, a.alpha, a.alpha, a.alpha};
    if (a.gate != nullptr) k *= reinterpret_cast<const floatx4 *>(a.gate)[c];
    if (post) k *= reinterpret_cast<const floatx4 *>(a.w_post)[c];
    return k;
  };
  floatx4 wp[kKeep ? kChunks : 1], wk[kKeep ? kChunks : 1];
  if constexpr (kKeep) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (int)threadIdx.x + i * threads;
      wp[i] = wk[i] = zero;
      if (c < a.chunks) {
        wp[i] = reinterpret_cast<const floatx4 *>(a.w_pre)[c];
        wk[i] = weight_k(c);
      }
    }
  }
  u32x2 hn[kChunks];
  floatx4 rn[kChunks];
  auto load = [&](int64_t row) {
    const u32x2 *h = reinterpret_cast<const u32x2 *>(a.h) + row * a.chunks;
    const floatx4 *res = reinterpret_cast<const floatx4 *>(a.res) + row * a.chunks;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (int)threadIdx.x + i * threads;
      hn[i] = (u32x2){0u, 0u};
      rn[i] = zero;
      if (c < a.chunks) {
        hn[i] = __builtin_nontemporal_load(h + c);
        rn[i] = __builtin_nontemporal_load(res + c);
      }
    }
  };
  if (kKeep && blockIdx.x < a.m) load(blockIdx.x);
  int turn = 0;
#pragma unroll 1
  for (int64_t row = blockIdx.x; row < a.m; row += gridDim.x) {
    const int64_t base = row * a.chunks;
    if constexpr (!kKeep) load(row);
    u32x2 hv[kChunks];
    floatx4 r[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      hv[i] = hn[i];
      r[i] = rn[i];
    }
    if (kKeep && row + gridDim.x < a.m) load(row + gridDim.x);
    float scale = 1.0f;
    if (post) {
      float sum[1] = {0.0f};
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const floatx4 v = bf16x4_values(hv[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[0] += v[j] * v[j];
      }
      row_block_sum(sum, part[turn]);
      turn ^= 1;
      const float rms = __builtin_sqrtf(sum[0] * inv_d + a.eps);
      if (threadIdx.x == 0) a.rms_post[row] = rms;
      scale = 1.0f / rms;
    }
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (int)threadIdx.x + i * threads;
      if (c < a.chunks) {
        const floatx4 k = kKeep ? wk[kKeep ? i : 0] : weight_k(c);
        r[i] += bf16x4_values(hv[i]) * scale * k;
        __builtin_nontemporal_store(r[i], reinterpret_cast<floatx4 *>(a.res_out) + base + c);
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[0] += r[i][j] * r[i][j];
      }
    }
    row_block_sum(sum, part[turn]);
    turn ^= 1;
    const float rms = __builtin_sqrtf(sum[0] * inv_d + a.eps);
    if (threadIdx.x == 0) a.rms_pre[row] = rms;
    const float inv = 1.0f / rms;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = (int)threadIdx.x + i * threads;
      if (c < a.chunks) {
        const floatx4 w = kKeep ? wp[kKeep ? i : 0] : reinterpret_cast<const floatx4 *>(a.w_pre)[c];
        const floatx4 o = r[i] * inv * w;
        __builtin_nontemporal_store(bf16x4_pack(o), reinterpret_cast<u32x2 *>(a.y) + base + c);
      }
    }
  }
}

struct BlockNormBwd {
  const uint16_t *dy;
  const float *dres;  // NULL: zero
  const float *res;   // r', or NULL with its checkpoint in codes and scales
  const uint32_t *codes;
  const float *scales;
  const float *rms_pre, *w_pre;
  const uint16_t *h;  // NULL: no block, y = norm(r') alone
  const float *rms_post, *w_post, *gate;
  float alpha;
  int64_t m;
  int32_t chunks, blocks;  // d / 4, checkpoint blocks a row
  int32_t row_threads;     // threads of a row; a workgroup may have several rows
  float *dres_out;         // may be dres
  uint16_t *dh;
  float *part;  // [G][2][d] column sums: dy r^, g h^
};

// What stays in registers between a row's sums and its outputs.
enum {
  kReload,  // nothing: both passes read the row and the weights
  kRow,     // the row
  kAhead,   // the row and the weights, with the next row on its way
};

// A row's operands, one chunk of four elements a thread.
struct NormChunk {
  floatx4 r;  // r', or its codes in r[0] and their scale in r[1]
  floatx4 g;  // dr'
  u32x2 dy, h;
};

// With f = 1 / rms_pre and q = 1 / rms_post the sums are taken over raw values,
//   A = f sum e r,  B = q sum k h (dr' + f e),  C = f q sum k h r,
// and the outputs from two factors a row: g = dr' + f e - (A / d) f^2 r and
// dh = q k g - (E / d) q^2 h, E = B - (A / d) f C: 21 vector instructions an
// element, which the waves of a SIMD (four up to 12288 columns) overlap with the
// memory.
template <int kMaxThreads, int kChunks, bool kH, int kMode>
__global__ void __launch_bounds__(kMaxThreads) block_norm_bwd_kernel(const BlockNormBwd a) {
  __shared__ float part[2][48];
  extern __shared__ floatx4 joined[];  // [2][chunks] where a workgroup has several rows
  const int tid = (int)threadIdx.x % a.row_threads;
  const int team = __builtin_amdgcn_readfirstlane((int)threadIdx.x / a.row_threads);
  const int teams = (int)blockDim.x / a.row_threads;
  const int threads = a.row_threads;
  const bool post = kH && a.w_post != nullptr;
  const float inv_d = 1.0f / (float)(4 * a.chunks);
  const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};

  auto weight_pre = [&](int c) { return reinterpret_cast<const floatx4 *>(a.w_pre)[c]; };
  auto weight_k = [&](int c) {
    floatx4 k = {a.alpha, a.alpha, a.alpha, a.alpha};
    if (a.gate != nullptr) k *= reinterpret_cast<const floatx4 *>(a.gate)[c];
    if (a.w_post != nullptr) k *= reinterpret_cast<const floatx4 *>(a.w_post)[c];
    return k;
  };
  constexpr bool kWeights = kMode == kAhead;
  floatx4 wp[kWeights ? kChunks : 1], wk[kWeights ? kChunks : 1];
  floatx4 sum_pre[kChunks], sum_h[kChunks];
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = tid + i * threads;
    sum_pre[i] = sum_h[i] = zero;
    if constexpr (kWeights) {
      wp[i] = wk[i] = zero;
      if (c < a.chunks) {
        wp[i] = weight_pre(c);
        if (kH) wk[i] = weight_k(c);
      }
    }
  }
  auto load = [&](int64_t row, int c) {
    NormChunk v;
    v.r = v.g = zero;
    v.dy = v.h = (u32x2){0u, 0u};
    if (row < a.m && c < a.chunks) {
      const int64_t at = row * a.chunks + c;
      if (a.res != nullptr) {
        v.r = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(a.res) + at);
      } else {
        v.r[0] = __builtin_bit_cast(float, a.codes[at]);
        v.r[1] = a.scales[row * a.blocks + (c >> kCkptBlockShift)];
      }
      if (a.dres != nullptr)
        v.g = __builtin_nontemporal_load(reinterpret_cast<const floatx4 *>(a.dres) + at);
      v.dy = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(a.dy) + at);
      if (kH) v.h = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(a.h) + at);
    }
    return v;
  };
  auto residual = [&](const NormChunk &v) {
    if (a.res != nullptr) return v.r;
    const float codes = v.r[0];
    return ckpt_values(__builtin_bit_cast(uint32_t, codes), v.r[1]);
  };
  auto fma4 = [](const floatx4 &x, const floatx4 &y, const floatx4 &z) {
    return __builtin_elementwise_fma(x, y, z);
  };
  auto all = [](float v) { return (floatx4){v, v, v, v}; };

  constexpr bool kHold = kMode != kReload;
  constexpr int kHeld = kHold ? kChunks : 1;
  auto load_row = [&](NormChunk (&v)[kHeld], int64_t row) {
    if constexpr (kHold) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) v[i] = load(row, tid + i * threads);
    }
  };
  auto work = [&](NormChunk (&v)[kHeld], int64_t row, float *sums) {
    const bool here = row < a.m;
    const float f = here ? 1.0f / a.rms_pre[row] : 0.0f;
    const float q = here && post ? 1.0f / a.rms_post[row] : 1.0f;
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = tid + i * threads;
      const bool in = c < a.chunks;
      const NormChunk x = kHold ? v[kHold ? i : 0] : load(row, c);
      const floatx4 p = kWeights ? wp[kWeights ? i : 0] : in ? weight_pre(c) : zero;
      const floatx4 r = residual(x), e = bf16x4_values(x.dy) * p;
#pragma unroll
      for (int j = 0; j < 4; ++j) s[0] = __builtin_fmaf(e[j], r[j], s[0]);
      if (post) {
        const floatx4 k = kWeights ? wk[kWeights ? i : 0] : in ? weight_k(c) : zero;
        const floatx4 kh = bf16x4_values(x.h) * k;
        const floatx4 b = fma4(e, all(f), x.g);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[1] = __builtin_fmaf(kh[j], b[j], s[1]);
          s[2] = __builtin_fmaf(kh[j], r[j], s[2]);
        }
      }
    }
    row_team_sum(s, sums, team, threads >> 6);
    if constexpr (kHold) {
      // Opaque: products and conversions of the first pass are made again rather
      // than held.
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        asm volatile("" : "+v"(v[i].r), "+v"(v[i].dy), "+v"(v[i].h));
    }
    if (!here) return;
    const float mean = s[0] * f * inv_d;                               // A / d
    const float mean_post = (s[1] - mean * f * f * s[2]) * q * inv_d;  // E / d
    const float cr = -mean * f * f, ch = -mean_post * q * q;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int c = tid + i * threads;
      if (c >= a.chunks) continue;
      const NormChunk x = kHold ? v[kHold ? i : 0] : load(row, c);
      const floatx4 p = kWeights ? wp[kWeights ? i : 0] : weight_pre(c);
      const floatx4 r = residual(x), dy = bf16x4_values(x.dy);
      const floatx4 t = fma4(r, all(cr), fma4(dy * p, all(f), x.g));
      sum_pre[i] = fma4(dy * f, r, sum_pre[i]);
      const int64_t at = row * a.chunks + c;
      __builtin_nontemporal_store(t, reinterpret_cast<floatx4 *>(a.dres_out) + at);
      if constexpr (kH) {
        const floatx4 k = kWeights ? wk[kWeights ? i : 0] : weight_k(c);
        const floatx4 h = bf16x4_values(x.h);
        sum_h[i] = fma4(t * q, h, sum_h[i]);
        floatx4 o = t * k;
        if (post) o = fma4(h, all(ch), o * q);
        __builtin_nontemporal_store(bf16x4_pack(o), reinterpret_cast<u32x2 *>(a.dh) + at);
      }
    }
  };

  // Every team of a workgroup takes as many rows, those past the last as zeros.
  const int64_t stride = (int64_t)gridDim.x * teams;
  int64_t row = (int64_t)blockIdx.x * teams;  // the first team's
  NormChunk v0[kHeld], v1[kHeld];
  if (kMode == kAhead) load_row(v0, row + team);
#pragma unroll 1
  for (; row < a.m; row += 2 * stride) {
    if (kMode == kAhead)
      load_row(v1, row + stride + team);
    else
      load_row(v0, row + team);
    work(v0, row + team, part[0]);
    if (row + stride >= a.m) break;
    if (kMode == kAhead) {
      load_row(v0, row + 2 * stride + team);
      work(v1, row + stride + team, part[1]);
    } else {
      load_row(v0, row + stride + team);
      work(v0, row + stride + team, part[1]);
    }
  }

  // The other teams' sums into the first's, one after the other.
  for (int t = 1; t < teams; ++t) {
    __syncthreads();
    if (team == t) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = tid + i * threads;
        if (c < a.chunks) {
          joined[c] = sum_pre[i];
          if (kH) joined[a.chunks + c] = sum_h[i];
        }
      }
    }
    __syncthreads();
    if (team == 0) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = tid + i * threads;
        if (c < a.chunks) {
          sum_pre[i] += joined[c];
          if (kH) sum_h[i] += joined[a.chunks + c];
        }
      }
    }
  }
  if (team != 0) return;
  floatx4 *out = reinterpret_cast<floatx4 *>(a.part) + (int64_t)blockIdx.x * 2 * a.chunks;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int c = tid + i * threads;
    if (c < a.chunks) {
      out[c] = sum_pre[i];
      if (kH) out[a.chunks + c] = sum_h[i];
    }
  }
}

// Adds the workgroups' column sums in order: a workgroup takes 16 chunks of
// columns, its 16 row groups each every 16th partial, joined through LDS.
__global__ void __launch_bounds__(256) block_norm_columns_kernel(
    const float *part, int32_t parts, int32_t chunks, const float *w_post, const float *gate,
    float alpha, float *dw_pre, float *dw_post, float *dgate) {
  __shared__ floatx4 lds[16][16];
  const int lane = threadIdx.x & 15, group = threadIdx.x >> 4;
  const int per = (chunks + 15) / 16;
  const int which = (int)blockIdx.x / per;  // 0: dy r^, 1: g h^
  const int c = ((int)blockIdx.x - which * per) * 16 + lane;
  floatx4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < chunks) {
    const floatx4 *p = reinterpret_cast<const floatx4 *>(part) + (int64_t)which * chunks + c;
#pragma unroll 8
    for (int i = group; i < parts; i += 16) s += p[(int64_t)i * 2 * chunks];
  }
  lds[group][lane] = s;
  __syncthreads();
  if (group != 0 || c >= chunks) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += lds[i][lane];
  if (which == 0) {
    reinterpret_cast<floatx4 *>(dw_pre)[c] = s;
    return;
  }
  s *= alpha;
  if (dw_post != nullptr) {
    floatx4 v = s;
    if (gate != nullptr) v *= reinterpret_cast<const floatx4 *>(gate)[c];
    reinterpret_cast<floatx4 *>(dw_post)[c] = v;
  }
  if (dgate != nullptr) {
    floatx4 v = s;
    if (w_post != nullptr) v *= reinterpret_cast<const floatx4 *>(w_post)[c];
    reinterpret_cast<floatx4 *>(dgate)[c] = v;
  }
}

// Waves of the persistent forward on a CU.
constexpr int kFwdWaves = 8;

// Threads of a row of `chunks` chunks: four chunks a thread up to 1024 threads,
// then eight.
static int row_chunks_per_thread(int64_t chunks) { return chunks <= 4096 ? 4 : 8; }
static int row_threads(int64_t chunks) {
  const int64_t per = row_chunks_per_thread(chunks);
  return (int)(((chunks + per - 1) / per + 63) / 64 * 64);
}

// The backward holds more a thread: up to 8192 elements 2 chunks and the next
// row (8192 rows of 8192: 219 us; 4 chunks on half as many threads 222, without
// the next row 253), up to 12288 3 chunks (with the next row only without a
// block, whose registers it takes; 4096 rows of 12288: 206 us, 427 with the next
// row, 259 with 8 chunks), up to 16384 8 chunks on half as many threads, then 8
// on 1024 and the row read twice.
static int bwd_threads(int64_t chunks) {
  const int64_t per = chunks <= 2048 ? 2 : (chunks <= 3072 ? 3 : 8);
  return (int)(((chunks + per - 1) / per + 63) / 64 * 64);
}

// Waves of the backward that a CU holds: two a SIMD of the kernel of 12292 to
// 16384 columns, which takes up to 256 registers, four of the others.  (1000 rows
// of 16384: 84 us; with 16 waves, twice the workgroups in two rounds, 94.)
static int bwd_waves(int64_t chunks) { return chunks > 3072 && chunks <= 4096 ? 8 : 16; }

// Rows of a backward workgroup side by side: up to 512 threads.
static int bwd_teams(int64_t chunks) {
  const int t = bwd_threads(chunks);
  return t >= 512 ? 1 : 512 / t;
}

// Workgroups of the backward: at most as many as run at once (bwd_waves).
// Every one writes two rows of column sums, so one row a team only up to one
// workgroup a CU, then two (64 rows of 4096: 9.5 us with one row a team, 13.1
// with four; 512 rows: 16.0 us with two, 21.3 with one).
static int64_t bwd_groups(int64_t m, int64_t d) {
  const int64_t teams = bwd_teams(d / 4), waves = teams * (bwd_threads(d / 4) / 64);
  const int64_t cus = cu_slots(), fit = bwd_waves(d / 4);
  const int64_t most = cus * (waves >= fit ? 1 : fit / waves);
  const int64_t one = (m + teams - 1) / teams, two = (m + 2 * teams - 1) / (2 * teams);
  const int64_t n = one < cus ? one : (two > cus ? two : cus);
  return n < most ? n : most;
}

static int32_t row_shape(int64_t m, int64_t d) {
  if (m < 0 || d <= 0)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "bad block norm shape m=%lld d=%lld", (long long)m,
                (long long)d);
  if (d % 4 != 0)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "block norm needs d %% 4 == 0, got %lld",
                (long long)d);
  if (d > kMaxRow)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "block norm row of %lld elements is too long",
                (long long)d);
  if (m > kMaxThreadsPerLaunch / 1024)
    return fail(NF4S_ERR_UNSUPPORTED_SHAPE, "too many rows");
  return NF4S_OK;
}

}  // namespace nf4s

using namespace nf4s;

extern "C" {

int32_t nf4s_block_norm_fwd(const uint16_t *h, const float *res, const float *w_pre,
                            const float *w_post, const float *gate, float alpha, int64_t m,
                            int64_t d, float eps, float *res_out, uint16_t *y, float *rms_pre,
                            float *rms_post, void *stream) {
  clear_error();
  const int32_t rc = row_shape(m, d);
  if (rc != NF4S_OK || m == 0) return rc;
  if (h == nullptr || res == nullptr || w_pre == nullptr || res_out == nullptr || y == nullptr ||
      rms_pre == nullptr || (w_post != nullptr && rms_post == nullptr))
    return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
  if (!aligned(res, 16) || !aligned(w_pre, 16) || !aligned(w_post, 16) || !aligned(gate, 16) ||
      !aligned(res_out, 16) || !aligned(h, 8) || !aligned(y, 8) || !aligned(rms_pre, 4) ||
      !aligned(rms_post, 4))
    return fail(NF4S_ERR_MISALIGNED,
                "block norm: fp32 rows and weights must be 16-byte aligned, h and y 8-byte");
  const BlockNormFwd a{h,   res, w_pre, w_post, gate, alpha, eps, m, (int32_t)(d / 4), res_out,
                       y,   rms_pre, rms_post};
  const int threads = row_threads(d / 4);
  auto *kernel = row_chunks_per_thread(d / 4) == 8 ? block_norm_fwd_kernel<1024, 8, false>
                 : threads <= 512                  ? block_norm_fwd_kernel<512, 4, true>
                                                   : block_norm_fwd_kernel<1024, 4, true>;
  const int wgs = threads >= 64 * kFwdWaves ? 1 : 64 * kFwdWaves / threads;
  const int64_t most = (int64_t)cu_slots() * wgs;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)(m < most ? m : most)), dim3(threads), 0,
                     as_stream(stream), a);
  return check_launch("block_norm_fwd_kernel");
}

int32_t nf4s_block_norm_bwd_workspace_size(int64_t m, int64_t d, int64_t *bytes) {
  clear_error();
  if (bytes == nullptr) return fail(NF4S_ERR_INVALID_ARGUMENT, "bytes is NULL");
  *bytes = 0;
  const int32_t rc = row_shape(m, d);
  if (rc != NF4S_OK) return rc;
  *bytes = bwd_groups(m, d) * 2 * d * 4;
  return NF4S_OK;
}

int32_t nf4s_block_norm_bwd(const uint16_t *dy, const float *dres, const float *res,
                            const uint8_t *res_codes, const float *res_scales, const float *rms_pre,
                            const float *w_pre, const uint16_t *h, const float *rms_post,
                            const float *w_post, const float *gate, float alpha, int64_t m,
                            int64_t d, float *dres_out, uint16_t *dh, float *dw_pre,
                            float *dw_post, float *dgate, void *workspace,
                            int64_t workspace_bytes, void *stream) {
  clear_error();
  const int32_t rc = row_shape(m, d);
  if (rc != NF4S_OK) return rc;
  if (w_pre == nullptr || dw_pre == nullptr)
    return fail(NF4S_ERR_INVALID_ARGUMENT, "w_pre or dw_pre is NULL");
  if ((w_post != nullptr) != (dw_post != nullptr) || (gate != nullptr) != (dgate != nullptr))
    return fail(NF4S_ERR_INVALID_ARGUMENT,
                "dw_post goes with w_post, and dgate with gate: both or neither");
  if (!aligned(w_pre, 16) || !aligned(w_post, 16) || !aligned(gate, 16) || !aligned(dw_pre, 16) ||
      !aligned(dw_post, 16) || !aligned(dgate, 16))
    return fail(NF4S_ERR_MISALIGNED, "block norm: weights and their gradients must be 16-byte "
                                     "aligned");
  const int64_t groups = bwd_groups(m, d);
  if (m > 0) {
    const bool coded = res_codes != nullptr;
    if (dy == nullptr || rms_pre == nullptr || dres_out == nullptr)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "NULL buffer");
    if (coded == (res != nullptr) || coded != (res_scales != nullptr))
      return fail(NF4S_ERR_INVALID_ARGUMENT,
                  "exactly one of res and res_codes with res_scales must be set");
    if ((h != nullptr) != (dh != nullptr))
      return fail(NF4S_ERR_INVALID_ARGUMENT, "dh goes with h: both or neither");
    if (h == nullptr && (w_post != nullptr || gate != nullptr))
      return fail(NF4S_ERR_INVALID_ARGUMENT, "w_post and gate need h");
    if (w_post != nullptr && rms_post == nullptr)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "w_post needs rms_post");
    if (!aligned(dres, 16) || !aligned(res, 16) || !aligned(dres_out, 16) || !aligned(dy, 8) ||
        !aligned(h, 8) || !aligned(dh, 8) || !aligned(res_codes, 4) || !aligned(res_scales, 4) ||
        !aligned(rms_pre, 4) || !aligned(rms_post, 4))
      return fail(NF4S_ERR_MISALIGNED,
                  "block norm: fp32 rows must be 16-byte aligned, dy, h and dh 8-byte");
    if (workspace == nullptr || workspace_bytes < groups * 2 * d * 4)
      return fail(NF4S_ERR_INVALID_ARGUMENT, "block norm backward needs %lld workspace bytes",
                  (long long)(groups * 2 * d * 4));
    if (!aligned(workspace, 16))
      return fail(NF4S_ERR_MISALIGNED, "workspace must be 16-byte aligned");
  }
  const hipStream_t s = as_stream(stream);
  const int32_t chunks = (int32_t)(d / 4);
  if (m > 0) {
    const BlockNormBwd a{dy,
                         dres,
                         res,
                         reinterpret_cast<const uint32_t *>(res_codes),
                         res_scales,
                         rms_pre,
                         w_pre,
                         h,
                         rms_post,
                         w_post,
                         gate,
                         alpha,
                         m,
                         chunks,
                         (int32_t)((d + kCkptBlock - 1) / kCkptBlock),
                         bwd_threads(chunks),
                         dres_out,
                         dh,
                         static_cast<float *>(workspace)};
    const int threads = bwd_threads(chunks);
    const bool blk = h != nullptr;
    auto *kernel = blk ? block_norm_bwd_kernel<1024, 2, true, kAhead>
                       : block_norm_bwd_kernel<1024, 2, false, kAhead>;
    if (chunks > 4096)
      kernel = blk ? block_norm_bwd_kernel<1024, 8, true, kReload>
                   : block_norm_bwd_kernel<1024, 8, false, kReload>;
    else if (chunks > 2048 && chunks <= 3072)
      kernel = blk ? block_norm_bwd_kernel<1024, 3, true, kRow>
                   : block_norm_bwd_kernel<1024, 3, false, kAhead>;
    else if (chunks > 3072)
      kernel = blk ? block_norm_bwd_kernel<512, 8, true, kRow>
                   : block_norm_bwd_kernel<512, 8, false, kRow>;
    const int teams = bwd_teams(chunks);
    hipLaunchKernelGGL(kernel, dim3((uint32_t)groups), dim3(threads * teams),
                       teams > 1 ? (uint32_t)(32 * chunks) : 0, s, a);
    const int32_t rc2 = check_launch("block_norm_bwd_kernel");
    if (rc2 != NF4S_OK) return rc2;
  }
  // Over no rows the sums are zero.
  const bool along = dw_post != nullptr || dgate != nullptr;
  hipLaunchKernelGGL(block_norm_columns_kernel, dim3((chunks + 15) / 16 * (along ? 2 : 1)),
                     dim3(256), 0, s, static_cast<const float *>(workspace), (int32_t)groups,
                     chunks, w_post, gate, alpha, dw_pre, dw_post, dgate);
  return check_launch("block_norm_columns_kernel");
}

}  // extern "C"
