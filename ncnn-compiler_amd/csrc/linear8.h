// Products of tokens in 8-bit integers as their kernels see them (linear8.hip,
// linear8_tiles.hip).
#pragma once

#include "elem.h"

namespace nhip {

// Codes, of tokens and of weights, lie as the matrix instructions take them:
// [rows / 16][steps][4][16 rows][16 codes], a step being 64 of the summed index
// and 1 KB of 16 rows.  What is past the rows or the sum is 0.  (Copies of rows
// of 64 bytes from codes in the tokens' own order ran at a quarter of the rate of
// whole kilobytes: 38 and 145 GB/s into the LDS of a CU.)
constexpr int kStepK = 64;
__host__ __device__ inline int64_t code_at(int64_t row, int steps) { return (row >> 4) * steps * 1024 + (row & 15) * 16; }

struct Linear8Args {
  const int8_t* x;       // codes of [rows]
  const float* x_scale;  // [rows]
  const int8_t* w;       // codes of [experts][16 blocks]
  const float* w_scale;  // [experts][n]
  const float* bias;     // [experts][n]
  void* out;             // [rows][n]
  const int32_t* starts;  // [experts + 1], or null: one expert, all rows
  int32_t rows, n, steps, blocks, experts, act;
};

// Rows of an expert, inside 0 .. rows - 1 whatever the starts say.
__device__ __forceinline__ void expert_rows(const Linear8Args& a, int e, int& begin, int& end) {
  begin = 0;
  end = a.rows;
  if (a.starts) {
    begin = max(0, min(a.starts[e], a.rows));
    end = max(begin, min(a.starts[e + 1], a.rows));
  }
}

// The sum of a product of codes as the result.
template <int ACT>
__device__ __forceinline__ float finish8(int sum, float x_scale, float w_scale, float bias) {
  const float y = fmaf((float)sum, x_scale * w_scale, bias);
  if constexpr (ACT == NHIP_ACT_RELU) return y < 0.f ? 0.f : y;  // NaN stays
  if constexpr (ACT == NHIP_ACT_SILU) return y * __builtin_amdgcn_rcpf(1.f + __expf(-y));
  return y;
}

// Calls `f` with the activation as a constant.
#define NHIP_FOR_ACT(act, ACT, ...)              \
  [&]() -> int {                                 \
    switch (act) {                               \
      case NHIP_ACT_RELU: {                      \
        constexpr int ACT = NHIP_ACT_RELU;       \
        return __VA_ARGS__;                      \
      }                                          \
      case NHIP_ACT_SILU: {                      \
        constexpr int ACT = NHIP_ACT_SILU;       \
        return __VA_ARGS__;                      \
      }                                          \
      default: {                                 \
        constexpr int ACT = NHIP_ACT_NONE;       \
        return __VA_ARGS__;                      \
      }                                          \
    }                                            \
  }()

// Integer sums on their way out of the matrix instructions, before any branch:
// the compiler's count of the cycles to wait was seen to miss the path on which
// a branch is taken.
template <class V>
__device__ __forceinline__ void settle8(V& sums) {
  asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sums));
}

bool linear8_tiles_selected(const Linear8Args& a);
int linear8_tiles(const Linear8Args& a, int dtype, hipStream_t s);

}  // namespace nhip
