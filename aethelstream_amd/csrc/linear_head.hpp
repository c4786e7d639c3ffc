// linear_head.hpp - what the operators over the logits of a linear head share:
// cross entropy (linear_ce.hip) and log probabilities (linear_logprob.hip).  Tiles
// of the logits, pieces of the vocabulary and the products of the gradients are
// chosen and launched in linear_ce.hip.
#pragma once

#include "bf16_gemm_core.hpp"

namespace nf4s {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Tokens of one forward launch, which bounds its partial sums.
constexpr int64_t kCeTokens = 16384;
// A launch counts its threads in 32 bits.
constexpr int64_t kMaxTiles = 0xffffffffll / kGcThreads;

// Maximum and sum of exponentials of part of a token's logits.
typedef float floatx2 __attribute__((ext_vector_type(2)));

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

// Tile columns of a strip (gc_tile): 4096 x 32000 x 8192 forward 1520 us with 4,
// 1549 with 6, 1577 with 8, 1666 with 16.
constexpr int kCeStrip = 4;

inline int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// A logits launch: 64 mt x 64 nt tiles over the next `cols` columns.
struct CeLaunch {
  int mt, nt;
  int64_t cols;
};

inline int64_t ceil_to(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct CePlan {
  int64_t tokens;        // forward: tokens of one launch
  int64_t part_bytes, fwd_bytes;
  int64_t piece, ldg;    // backward: columns of a piece, row length of G
  int dx_mt;
  int64_t slices, slice; // of dx's reduction over a piece
  int64_t g_bytes, bwd_bytes;
};


// Launches over the tiles of m > 0 tokens by v > 0 columns: one or two.
int ce_tiles(int64_t m, int64_t v, int64_t d, CeLaunch (&out)[2]);
// Partial sums a token leaves: one for each half tile.
int64_t ce_slices(int64_t m, int64_t v, int64_t d);
int32_t ce_plan(int64_t m, int64_t v, int64_t d, CePlan &p);
// Checks what both directions read, and a workspace of `need` bytes.
int32_t ce_operands(const uint16_t *x, const uint16_t *w, const int64_t *targets, int64_t m,
                    void *workspace, int64_t workspace_bytes, int64_t need);

// Gradients of a function of the logits, whose own gradient G is made by pieces.
struct HeadGrad {
  const uint16_t *x, *w;
  int64_t m, v, d;
  uint16_t *dx;
  void *dw;
  bool dw_is_f32, accumulate;
  void *workspace;  // CePlan::bwd_bytes
};
// A piece of G: columns v0 .. v0 + vn - 1 of the vocabulary, rows ldg long with
// zeros from vn on, divided by *common.
struct HeadPiece {
  int64_t v0, vn;
  uint16_t *g;
  int64_t ldg;
  const float *common;
  hipStream_t stream;
};
typedef int32_t (*HeadLogits)(const void *ctx, const HeadPiece &);

// Where the factor that all of G is divided by stands: set before the pieces.
inline float *head_common(const HeadGrad &h, const CePlan &p) {
  return reinterpret_cast<float *>(static_cast<char *>(h.workspace) + p.g_bytes) +
         p.slices * h.m * h.d;
}
int32_t head_gradients(const HeadGrad &h, const CePlan &p, HeadLogits logits, const void *ctx,
                       hipStream_t s);
// dw over no tokens.
int32_t head_zero_dw(void *dw, bool f32, int64_t n, hipStream_t s);

}  // namespace nf4s
