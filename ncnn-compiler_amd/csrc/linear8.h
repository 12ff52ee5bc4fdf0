// Products of tokens in 8-bit integers as their kernels see them (linear8.hip,
// linear8_tiles.hip).
#pragma once

#include "elem.h"

namespace nhip {

// Operands are walked in steps of 64 of the summed index, two at a time: rows of
// codes are padded to a multiple of kPadK, with zeros.
constexpr int kStepK = 64, kPadK = 128;

// The weights of one expert lie as the matrix instructions take them:
// [n / 16][k / 64][4][16 rows][16 codes], 1 KB to 16 rows and 64 codes.
struct Linear8Args {
  const int8_t* x;       // codes [rows][kp]
  const float* x_scale;  // [rows]
  const int8_t* w;       // [experts][blocks][steps][1024]
  const float* w_scale;  // [experts][n]
  const float* bias;     // [experts][n]
  void* out;             // [rows][n]
  const int32_t* starts;  // [experts + 1], or null: one expert, all rows
  int32_t rows, n, kp, steps, blocks, experts, act;
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
__device__ __forceinline__ float finish8(int sum, float scale, float bias) {
  const float y = (float)sum * scale + bias;
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
