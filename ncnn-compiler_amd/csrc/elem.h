// Element types of the token operators (group norm into tokens, rotary
// positions, attention): fp32, fp16 and bf16 in memory, fp32 in registers.
#pragma once

#include "nhip_internal.h"

namespace nhip {

typedef _Float16 f16;
typedef __bf16 bf16;
typedef f16 v8h __attribute__((ext_vector_type(8)));
typedef bf16 v8b __attribute__((ext_vector_type(8)));
typedef float v8f __attribute__((ext_vector_type(8)));

inline int elem_size(int dtype) {
  switch (dtype) {
    case NHIP_DTYPE_F32: return 4;
    case NHIP_DTYPE_F16:
    case NHIP_DTYPE_BF16: return 2;
    default: return 0;
  }
}

inline bool aligned_to(const void* p, uint64_t bytes) { return reinterpret_cast<uint64_t>(p) % bytes == 0; }

// N consecutive elements: one 16-byte access (4 fp32 or 8 16-bit elements) or
// a single element.  The pointer is aligned to the whole access.  STREAM: a
// store that takes no place in the caches, of a result that is too large for
// them to hold it until its use.
template <class T, int N>
struct Vec {
  typedef T type __attribute__((ext_vector_type(N)));
  __device__ __forceinline__ static void load(const T* p, float (&x)[N]) {
    const type v = *reinterpret_cast<const type*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
  }
  template <bool STREAM = false>
  __device__ __forceinline__ static void store(T* p, const float (&x)[N]) {
    type v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
    if constexpr (STREAM)
      __builtin_nontemporal_store(v, reinterpret_cast<type*>(p));
    else
      *reinterpret_cast<type*>(p) = v;
  }
};
template <class T>
struct Vec<T, 1> {
  __device__ __forceinline__ static void load(const T* p, float (&x)[1]) { x[0] = (float)*p; }
  template <bool STREAM = false>
  __device__ __forceinline__ static void store(T* p, const float (&x)[1]) { *p = (T)x[0]; }
};
constexpr int64_t kStreamBytes = 64 << 20;  // results past this are stored with STREAM
template <class T>
constexpr int kVec = 16 / sizeof(T);

// Calls `f` with a value of the element type that `dtype` names.
#define NHIP_FOR_ELEM(dtype, T, ...)          \
  [&]() -> int {                              \
    switch (dtype) {                          \
      case NHIP_DTYPE_F32: {                  \
        typedef float T;                      \
        return __VA_ARGS__;                   \
      }                                       \
      case NHIP_DTYPE_F16: {                  \
        typedef ::nhip::f16 T;                \
        return __VA_ARGS__;                   \
      }                                       \
      default: {                              \
        typedef ::nhip::bf16 T;               \
        return __VA_ARGS__;                   \
      }                                       \
    }                                         \
  }()

}  // namespace nhip
