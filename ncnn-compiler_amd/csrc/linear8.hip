// Products of tokens with weights in 8-bit integers, a scale for each token and
// each output channel: the tokens' codes, the product for few rows, the entry
// points.  (The product for many rows: linear8_tiles.hip.)
//
// Compiled with -ffp-contract=off: a code is the rounding of one separately
// rounded product, so that it can be restated bit for bit.
#include <algorithm>
#include <new>

#include "linear8.h"

struct nhip_linear8_plan {
  int32_t experts, n, k, act, device;
  int32_t blocks, steps;  // of 16 channels, of 64 summed indices
  int8_t* w = nullptr;
  float* w_scale = nullptr;  // [experts][n], the bias behind it
};

namespace nhip {
namespace {

constexpr int kMaxK = 131072;  // 128 * 127 * 131072 < 2^31 (a weight may be -128)
constexpr int kMaxRows = 0x3fffff0;  // a wave to each in a launch of below 2^32 threads
constexpr float kLeastScale = 1.17549435e-38f;  // 2^-126: the reciprocal stays finite

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// Eight channels from c of a row; those at and past k are 0.  Rows begin at any
// element: the card loads 16 bytes from any address (3356 rows of 5789 fp32 an element
// at a time 74 us, so 25, aligned rows 24).
template <class T>
__device__ __forceinline__ void load8(const T* row, int c, int k, float (&x)[8]) {
  if (c + 8 <= k) {
    constexpr int V = kVec<T>;
    typedef typename Vec<T, V>::type Any __attribute__((aligned(sizeof(T))));
#pragma unroll
    for (int j = 0; j < 8; j += V) {
      const Any t = *reinterpret_cast<const Any*>(row + c + j);
#pragma unroll
      for (int i = 0; i < V; ++i) x[j + i] = (float)t[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = c + i < k ? (float)row[c + i] : 0.f;
  }
}

// A row's scale from its largest magnitude (infinite: the row holds an infinity or NaN,
// its codes are 0 and its results 0 * NaN), and what x is multiplied by.
struct RowScale {
  float scale, inv;
  __device__ __forceinline__ explicit RowScale(float most) {
    scale = most > 0.f ? fmaxf(most * (1.f / 127.f), kLeastScale) : 0.f;
    inv = scale > 0.f && most < INFINITY ? 1.f / scale : 0.f;
    if (!(most < INFINITY)) scale = NAN;
  }
};
struct Widest {
  float most = 0.f;
  bool whole = true;  // finite
  __device__ __forceinline__ void show(const float (&t)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      most = fmaxf(most, fabsf(t[i]));
      whole = whole && fabsf(t[i]) <= 3.4028235e38f;
    }
  }
  __device__ __forceinline__ RowScale of_wave() const { return RowScale(wave_max(whole ? most : INFINITY)); }
};
__device__ __forceinline__ uint2 codes8(const float (&t)[8], float inv) {
  int q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = quantize_q(t[i], inv);
  return make_uint2(pack_i8x4(q[0], q[1], q[2], q[3]), pack_i8x4(q[4], q[5], q[6], q[7]));
}

// One workgroup: 8 rows, one to a wave, which finds its largest magnitude first;
// the codes are put in order in LDS, kChunk of a row at a time, and stored as the
// 128 bytes that 8 rows have together.  The first chunk is held, others are read again.
// Bytes bound it, at sizes like these with a launch's start and end beside them: 6272
// rows of 2048 bf16 11 us (39 MB, 3.5 TB/s), 12544 of 1024 fp16 12.5.
constexpr int kChunk = 2048;
template <class T>
__global__ __launch_bounds__(512) void linear8_codes_kernel(const T* x, int64_t stride, int rows, int k, int steps,
                                                             int8_t* codes, float* scales) {
  constexpr int HELD = kChunk / 8 / 64, ROW = kChunk + 16;  // (a row's chunks of 16 codes begin in different banks)
  __shared__ __attribute__((aligned(16))) int8_t lds[8 * ROW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = blockIdx.x * 8 + wave;
  const int mine = r < rows ? k : 0;  // past the rows: zeros
  const T* row = x + (int64_t)min(r, rows - 1) * stride;
  float held[HELD][8];
  Widest widest;
#pragma unroll
  for (int h = 0; h < HELD; ++h) load8<T>(row, (lane + h * 64) * 8, mine, held[h]);
#pragma unroll
  for (int h = 0; h < HELD; ++h) widest.show(held[h]);
#pragma unroll 4
  for (int c = kChunk + lane * 8; c < mine; c += 512) {
    float t[8];
    load8<T>(row, c, mine, t);
    widest.show(t);
  }
  const RowScale scale = widest.of_wave();
  if (lane == 0 && r < rows) scales[r] = scale.scale;
  int8_t* to = codes + code_at((int64_t)blockIdx.x * 8, steps);
  for (int c0 = 0; c0 < steps * kStepK; c0 += kChunk) {
    const int width = min(kChunk, steps * kStepK - c0);
    if (c0) __syncthreads();
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int c = (lane + h * 64) * 8;
      if (c >= width) break;
      if (c0) load8<T>(row, c0 + c, mine, held[h]);
      *reinterpret_cast<uint2*>(lds + wave * ROW + c) = codes8(held[h], scale.inv);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < width / 2; i += 512)  // 16 codes of a row: [steps][4][16 rows]
      *reinterpret_cast<int4*>(to + (int64_t)c0 * 16 + (i >> 3) * 256 + (i & 7) * 16) =
          *reinterpret_cast<const int4*>(lds + (i & 7) * ROW + (i >> 3) * 16);
  }
}

template <class T>
int codes_run(const void* x, int64_t stride, int64_t rows, int k, int steps, int8_t* codes, float* scales, hipStream_t s) {
  NHIP_LAUNCH("linear8_codes", linear8_codes_kernel<T>, dim3((uint32_t)ceil_div(rows, 16) * 2), dim3(512), 0, s, (const T*)x, stride,
              (int)rows, k, steps, codes, scales);
  return check_launch("linear8_codes");
}

// Codes [experts][n][k] in order, 16 codes to a thread.
__global__ __launch_bounds__(256) void linear8_order_kernel(const int8_t* from, int experts, int n, int k, int blocks, int steps,
                                                            bool vec, int8_t* to) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (item >= (int64_t)experts * blocks * steps * 64) return;
  const int lane = item & 63;
  int64_t at = item >> 6;
  const int step = (int)(at % steps);
  at /= steps;
  const int row = (int)(at % blocks) * 16 + (lane & 15), c = step * kStepK + (lane >> 4) * 16;
  int4 v = make_int4(0, 0, 0, 0);
  if (row < n && c < k) {
    const int8_t* src = from + (at / blocks * n + row) * k + c;
    if (vec && c + 16 <= k) {
      v = *reinterpret_cast<const int4*>(src);
    } else {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (c + i < k) w[i >> 2] |= (uint32_t)(uint8_t)src[i] << (8 * (i & 3));
      v = make_int4(w[0], w[1], w[2], w[3]);
    }
  }
  *reinterpret_cast<int4*>(to + item * 16) = v;
}

__global__ __launch_bounds__(256) void linear8_params_kernel(const float* scale, const float* bias, int64_t count,
                                                             float* to) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  if (scale) to[i] = scale[i];
  to[count + i] = bias ? bias[i] : 0.f;
}

// ---------------------------------------------------------------- few rows
// One workgroup: NB blocks of 16 channels of one expert, 16 TG of its rows, and if
// the expert has more than its share the rows `chunks` times as far on; its waves take
// the steps of the sum in turn and are joined in LDS.  Weights go from memory to the
// registers that the products read, every wave's next kAhead steps under way at a time.
// Reading them bounds it: 48 rows of 2048 to 50021 fp16 27 us for 102 MB (3.8 TB/s; a
// large copy 5.1) and 5 for the codes; where an expert has few rows, latency (128 rows of
// 16 experts, 2048 to 1024 12.1 us, 34 MB).
constexpr int kAhead = 4;  // steps that a wave reads before it multiplies them
// Weights take no place in the caches where each is read once.  With more than 48 rows
// to an expert others read them too, or the next to it: us past the caches / through
// them, three layers in turn, 64 rows of 4096 to 16384 25.9 / 24.4, 319 of 1920 over 6
// experts to 7488 36.7 / 31.4, 1200 of 8192 to 528 34.8 / 25.7; 48 of 2048 to 50021 31.2 / 32.9.
template <bool ONCE>
__device__ __forceinline__ v4i load_w(const int8_t* w) {
  const v4i* const at = reinterpret_cast<const v4i*>(w);
  return ONCE ? __builtin_nontemporal_load(at) : *at;
}
template <class T, int ACT, int TG, int NB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void linear8_rows_kernel(Linear8Args a, int chunks) {
  __shared__ v4i part[WAVES][TG * NB][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int groups = (a.blocks + NB - 1) / NB;
  const uint32_t of = blockIdx.x / groups;
  const int e = of / chunks, b0 = blockIdx.x % groups * NB;
  int begin, end;
  expert_rows(a, e, begin, end);
  const int8_t* w[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b)
    w[b] = a.w + ((int64_t)e * a.blocks + min(b0 + b, a.blocks - 1)) * a.steps * 1024 + lane * 16;
  for (int r0 = begin + of % chunks * (16 * TG); r0 < end; r0 += chunks * (16 * TG)) {
    const int8_t* x[TG];
#pragma unroll
    for (int t = 0; t < TG; ++t) x[t] = a.x + code_at(min(r0 + t * 16 + (lane & 15), end - 1), a.steps) + (lane >> 4) * 256;
    v4i acc[TG][NB];
#pragma unroll
    for (int t = 0; t < TG; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[t][b] = v4i{0, 0, 0, 0};
    for (int s = wave; s < a.steps; s += WAVES * kAhead) {
      v4i wf[kAhead][NB], xf[kAhead][TG];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int at = min(s + u * WAVES, a.steps - 1);
#pragma unroll
        for (int b = 0; b < NB; ++b) wf[u][b] = load_w<TG < 4>(w[b] + at * 1024);
#pragma unroll
        for (int t = 0; t < TG; ++t) xf[u][t] = *reinterpret_cast<const v4i*>(x[t] + at * 1024);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (s + u * WAVES >= a.steps)
#pragma unroll
          for (int b = 0; b < NB; ++b) wf[u][b] = v4i{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < TG; ++t)
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[t][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][b], xf[u][t], acc[t][b], 0, 0, 0);
      }
    }
#pragma unroll
    for (int t = 0; t < TG; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        settle8(acc[t][b]);
        part[wave][t * NB + b][lane] = acc[t][b];
      }
    __syncthreads();
    for (int i = threadIdx.x; i < TG * NB * 64; i += WAVES * 64) {
      v4i sum = part[0][i >> 6][i & 63];
#pragma unroll
      for (int v = 1; v < WAVES; ++v) sum += part[v][i >> 6][i & 63];
      const int l = i & 63, b = (i >> 6) % NB, t = (i >> 6) / NB;
      const int row = r0 + t * 16 + (l & 15), j = (b0 + b) * 16 + 4 * (l >> 4);
      if (row < end) {
        const float xs = a.x_scale[row];
        const float* ws = a.w_scale + (int64_t)e * a.n;
        const float* bias = a.bias + (int64_t)e * a.n;
        T* out = (T*)a.out + (int64_t)row * a.n;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (j + c < a.n) out[j + c] = (T)finish8<ACT>(sum[c], xs, ws[j + c], bias[j + c]);
      }
    }
    __syncthreads();
  }
}

// At most 16 rows in all, of at most kFewK, and few workgroups: each makes the codes
// itself, while the first weights are on their way, which spares a launch.  One block
// of 16 channels of one expert; the waves take the steps in turn.  Latency bounds it:
// 16 rows of 2048 to 2048 bf16 7.5 us a call (4 MB of weights: 0.8 at a large copy's
// rate), in two launches 10.0.
constexpr int kFewK = 2048;  // a row in the registers of a wave
template <class T, int ACT>
__global__ __launch_bounds__(512) void linear8_few_kernel(Linear8Args a, const T* x, int64_t stride, int k) {
  constexpr int WAVES = 8, HELD = kFewK / 8 / 64;
  __shared__ __attribute__((aligned(16))) int8_t codes[16 * kFewK];  // [steps][4][16 rows][16]
  __shared__ v4i part[WAVES][64];
  __shared__ float scales[16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int e = blockIdx.x / a.blocks, b = blockIdx.x % a.blocks;
  int begin, end;
  expert_rows(a, e, begin, end);
  if (begin >= end) return;
  const int8_t* w = a.w + ((int64_t)e * a.blocks + b) * a.steps * 1024 + lane * 16;
  v4i wf[kAhead];
#pragma unroll
  for (int u = 0; u < kAhead; ++u) wf[u] = *reinterpret_cast<const v4i*>(w + min(wave + u * WAVES, a.steps - 1) * 1024);
#pragma unroll
  for (int r = wave; r < 16; r += WAVES) {
    const int mine = begin + r < end ? k : 0;  // past the rows: zeros
    const T* row = x + (int64_t)min(begin + r, end - 1) * stride;
    float held[HELD][8];
    Widest widest;
#pragma unroll
    for (int h = 0; h < HELD; ++h) load8<T>(row, (lane + h * 64) * 8, mine, held[h]);
#pragma unroll
    for (int h = 0; h < HELD; ++h) widest.show(held[h]);
    const RowScale scale = widest.of_wave();
    if (lane == 0) scales[r] = scale.scale;
#pragma unroll
    for (int h = 0; h < HELD; ++h)
      if (const int c = (lane + h * 64) * 8; c < a.steps * kStepK)
        *reinterpret_cast<uint2*>(codes + (c >> 4) * 256 + r * 16 + (c & 8)) = codes8(held[h], scale.inv);
  }
  __syncthreads();
  v4i acc = {0, 0, 0, 0};
  for (int s = wave; s < a.steps; s += WAVES * kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = s + u * WAVES;
      if (at < a.steps)
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], *reinterpret_cast<const v4i*>(codes + at * 1024 + lane * 16), acc, 0, 0, 0);
      wf[u] = *reinterpret_cast<const v4i*>(w + min(at + WAVES * kAhead, a.steps - 1) * 1024);
    }
  }
  settle8(acc);
  part[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
#pragma unroll
  for (int v = 1; v < WAVES; ++v) acc += part[v][lane];
  const int row = begin + (lane & 15), j = b * 16 + 4 * (lane >> 4);
  if (row >= end) return;
  const float xs = scales[lane & 15];
  T* out = (T*)a.out + (int64_t)row * a.n;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (j + c < a.n) out[j + c] = (T)finish8<ACT>(acc[c], xs, a.w_scale[(int64_t)e * a.n + j + c], a.bias[(int64_t)e * a.n + j + c]);
}

// Every workgroup makes the codes of its rows again, which must not take longer than
// the launch that it spares.  us a call (one after the other, four layers in turn),
// this / in two launches, 16 rows bf16: 2048 to 2048 (128 workgroups) 9.0 / 12.0, to 8192
// (512) 10.7 / 12.6, to 12288 (768) 13.5 / 12.4, to 16384 17.4 / 12.6; 16 experts, 1024 to
// 512 (512) 9.6 / 12.5, 2048 to 1024 (1024) 17.4 / 12.5; with rows read twice, 4096 to 4096
// (256) 14.6 / 11.8, 8192 to 2048 (128) 24.0 / 18.5.
bool few_selected(const Linear8Args& a) {
  // (the switch that pins the other kernels pins them here too)
  if (a.rows > 16 || a.steps * kStepK > kFewK || setting_int("NHIP_LINEAR8_TILES", -1) >= 0) return false;
  return (int64_t)a.experts * a.blocks <= 2 * cu_count();
}

template <class T, int ACT>
int few_run(const Linear8Args& a, const void* x, int64_t stride, int k, hipStream_t s) {
  NHIP_LAUNCH("linear8_few", (linear8_few_kernel<T, ACT>), dim3((uint32_t)(a.experts * (int64_t)a.blocks)), dim3(512), 0, s, a, (const T*)x,
              stride, k);
  return check_launch("linear8_few");
}

template <class T, int ACT, int TG>
int rows_run(const Linear8Args& a, hipStream_t s) {
  const int64_t chunks = ceil_div(ceil_div(a.rows, a.experts), 16 * TG), wgs = a.experts * (int64_t)a.blocks * chunks;
  if (wgs > 0x1ffffff) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "linear8: too many tiles");
  const auto launch = [&](auto kernel, int nb, int waves) {
    NHIP_LAUNCH("linear8_rows", kernel, dim3((uint32_t)(a.experts * chunks * ceil_div(a.blocks, nb))), dim3(waves * 64), 0, s, a, (int)chunks);
    return check_launch("linear8_rows");
  };
  // us (NB, waves): 48 rows of 2048 to 50021 (3127 blocks) fp16 2, 2 31.8; 2, 4 33.4; 4, 4
  // 34.1; 1, 4 42.7; 128 rows of 16 experts, 2048 to 1024 (1024 blocks) bf16 2, 4 12.1; 1, 8
  // 13.2; 2, 2 13.4; 4, 4 15.0.
  if (wgs > 8 * cu_count()) return launch(linear8_rows_kernel<T, ACT, TG, 2, 2>, 2, 2);
  if (wgs > 2 * cu_count()) return launch(linear8_rows_kernel<T, ACT, TG, 2, 4>, 2, 4);
  return launch(linear8_rows_kernel<T, ACT, TG, 1, 8>, 1, 8);
}

template <class T, int ACT>
int product_run(const Linear8Args& a, hipStream_t s) {
  const int64_t each = ceil_div(a.rows, a.experts);
  if (each <= 16) return rows_run<T, ACT, 1>(a, s);
  if (each <= 32) return rows_run<T, ACT, 2>(a, s);
  if (each <= 48) return rows_run<T, ACT, 3>(a, s);
  return rows_run<T, ACT, 4>(a, s);
}

// Codes of the tokens, their scales behind them.
uint64_t workspace_of(const nhip_linear8_plan* p, int64_t rows) {
  return (uint64_t)round_up(rows, 16) * p->steps * kStepK + (uint64_t)round_up(rows * (int64_t)sizeof(float), 16);
}

// Whether any of the rows, `stride` bytes apart, holds a byte of `out`.
bool rows_meet(const void* x, int64_t rows, int64_t stride, int64_t row_bytes, const void* out, int64_t out_bytes) {
  const int64_t off = (int64_t)((uintptr_t)out - (uintptr_t)x);
  // the first row that ends behind the beginning of `out`
  const int64_t r = off < row_bytes ? 0 : stride ? (off - row_bytes) / stride + 1 : rows;
  return r < rows && r * stride < off + out_bytes;
}

int linear8_args(const nhip_linear8_plan* p, int32_t dtype, int64_t rows) {
  if (!p) return fail(NHIP_STATUS_NULL_POINTER, "linear8: null plan");
  if (!elem_size(dtype)) return fail(NHIP_STATUS_UNSUPPORTED, "linear8: dtype has to be F32, F16 or BF16");
  if (rows < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "linear8: negative extent");
  if (rows > kMaxRows) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "linear8: too many rows");
  return ok();
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int nhip_linear8_create(int32_t experts, int32_t num_output, int32_t num_input, const void* weight, int32_t weight_is_i8,
                        const float* weight_scale, const float* bias, int32_t activation, void* stream,
                        nhip_linear8_t* plan) {
  if (!plan) return fail(NHIP_STATUS_NULL_POINTER, "linear8: null plan pointer");
  *plan = nullptr;
  if (experts <= 0 || num_output <= 0 || num_input <= 0) return fail(NHIP_STATUS_INVALID_SHAPE, "linear8: sizes have to be positive");
  if (num_input > kMaxK) return fail(NHIP_STATUS_INVALID_SHAPE, "linear8: at most 131072 inputs, the sums are of 32 bits");
  if (activation != NHIP_ACT_NONE && activation != NHIP_ACT_RELU && activation != NHIP_ACT_SILU)
    return fail(NHIP_STATUS_UNSUPPORTED, "linear8: activation has to be NONE, RELU or SILU");
  const int64_t blocks = ceil_div(num_output, 16), steps = ceil_div(num_input, kStepK);
  if (num_output > kMaxRows || experts * blocks > 0x7fffffff / 4 || experts * (int64_t)num_output > 0x7fffffff)
    return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "linear8: too many output channels");
  if (!weight || (weight_is_i8 && !weight_scale)) return fail(NHIP_STATUS_NULL_POINTER, "linear8: null pointer");
  if (!weight_is_i8 && weight_scale)
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "linear8: scales come with 8-bit weights, those of fp32 weights are found here");
  if (!aligned_to(weight, weight_is_i8 ? 1 : 4) || !aligned_to(weight_scale, 4) || !aligned_to(bias, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "linear8: a tensor is not aligned to its type");
  const hipStream_t s = as_stream(stream);
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  NHIP_TRY(check_hip(hipStreamIsCapturing(s, &capture), "hipStreamIsCapturing"));
  if (capture != hipStreamCaptureStatusNone)
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "linear8: a plan is not made while the stream is recorded");
  nhip_linear8_plan* p = new (std::nothrow) nhip_linear8_plan;
  if (!p) return fail(NHIP_STATUS_DEVICE_ERROR, "linear8: out of host memory");
  p->experts = experts;
  p->n = num_output;
  p->k = num_input;
  p->act = activation;
  p->blocks = (int32_t)blocks;
  p->steps = (int32_t)steps;
  const int64_t count = experts * (int64_t)num_output, items = experts * blocks * steps * 64;
  const auto build = [&]() -> int {
    NHIP_TRY(check_hip(hipGetDevice(&p->device), "hipGetDevice"));
    if (items > 0xffffff00) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "linear8: too many weights");
    NHIP_TRY(check_hip(hipMalloc(reinterpret_cast<void**>(&p->w), items * 16), "hipMalloc(linear8 weights)"));
    NHIP_TRY(check_hip(hipMalloc(reinterpret_cast<void**>(&p->w_scale), 2 * count * sizeof(float)), "hipMalloc(linear8 scales)"));
    if (weight_is_i8) {
      NHIP_LAUNCH("linear8_order", linear8_order_kernel, dim3((uint32_t)ceil_div(items, 256)), dim3(256), 0, s,
                  (const int8_t*)weight, experts, num_output, num_input, (int)blocks, (int)steps,
                  aligned_to(weight, 16) && num_input % 16 == 0, p->w);
      NHIP_TRY(check_launch("linear8_order"));
    } else {
      for (int64_t e = 0; e < experts; ++e)
        NHIP_TRY(codes_run<float>((const float*)weight + e * num_output * num_input, num_input, num_output, num_input, (int)steps,
                                  p->w + e * blocks * steps * 1024, p->w_scale + e * num_output, s));
    }
    NHIP_LAUNCH("linear8_params", linear8_params_kernel, dim3((uint32_t)ceil_div(count, 256)), dim3(256), 0, s, weight_scale,
                bias, count, p->w_scale);
    NHIP_TRY(check_launch("linear8_params"));
    return check_hip(hipStreamSynchronize(s), "hipStreamSynchronize(linear8 plan)");
  };
  const int st = build();
  if (st != NHIP_STATUS_SUCCESS) {
    (void)hipFree(p->w);
    (void)hipFree(p->w_scale);
    delete p;
    return st;
  }
  *plan = p;
  return ok();
}

int nhip_linear8_workspace_size(nhip_linear8_t plan, int32_t dtype, int64_t rows, uint64_t* bytes) {
  if (!bytes) return fail(NHIP_STATUS_NULL_POINTER, "linear8: null pointer");
  NHIP_TRY(linear8_args(plan, dtype, rows));
  *bytes = rows ? workspace_of(plan, rows) : 0;
  return ok();
}

int nhip_linear8_forward(nhip_linear8_t plan, const void* x, int32_t dtype, int64_t rows, int64_t row_stride,
                         const int32_t* expert_starts, void* out, void* workspace, uint64_t workspace_bytes, void* stream) {
  NHIP_TRY(linear8_args(plan, dtype, rows));
  if (!expert_starts && plan->experts > 1)
    return fail(NHIP_STATUS_NULL_POINTER, "linear8: rows of several experts need their starts");
  if (rows == 0) return ok();
  if (!x || !out || !workspace) return fail(NHIP_STATUS_NULL_POINTER, "linear8: null pointer");
  const int es = elem_size(dtype);
  if (!aligned_to(x, es) || !aligned_to(out, es) || !aligned_to(expert_starts, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "linear8: a tensor is not aligned to its type");
  if (row_stride < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "linear8: negative stride");
  // (workgroups read tokens while others store results)
  if (rows_meet(x, rows, row_stride * es, (int64_t)plan->k * es, out, rows * plan->n * es))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "linear8: the results overlap the tokens");
  int dev = -1;
  NHIP_TRY(check_hip(hipGetDevice(&dev), "hipGetDevice"));
  if (dev != plan->device) return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "linear8: the plan is another device's");
  if (workspace_bytes < workspace_of(plan, rows) || !aligned_to(workspace, 16))
    return fail(NHIP_STATUS_OUTPUT_CAPACITY_INSUFFICIENT, "linear8: workspace too small or not 16-byte aligned");
  int8_t* codes = (int8_t*)workspace;
  float* scales = (float*)(codes + round_up(rows, 16) * plan->steps * kStepK);
  Linear8Args a{};
  a.x = codes;
  a.x_scale = scales;
  a.w = plan->w;
  a.w_scale = plan->w_scale;
  a.bias = plan->w_scale + plan->experts * (int64_t)plan->n;
  a.out = out;
  a.starts = expert_starts;
  a.rows = (int32_t)rows;
  a.n = plan->n;
  a.steps = plan->steps;
  a.blocks = plan->blocks;
  a.experts = plan->experts;
  a.act = plan->act;
  if (few_selected(a))
    return NHIP_FOR_ELEM(dtype, T, NHIP_FOR_ACT(a.act, ACT, few_run<T, ACT>(a, x, row_stride, plan->k, as_stream(stream))));
  NHIP_TRY(NHIP_FOR_ELEM(dtype, T, codes_run<T>(x, row_stride, rows, plan->k, plan->steps, codes, scales, as_stream(stream))));
  if (linear8_tiles_selected(a)) return linear8_tiles(a, dtype, as_stream(stream));
  return NHIP_FOR_ELEM(dtype, T, NHIP_FOR_ACT(a.act, ACT, product_run<T, ACT>(a, as_stream(stream))));
}

int nhip_linear8_destroy(nhip_linear8_t plan) {
  if (!plan) return ok();
  (void)hipFree(plan->w);
  (void)hipFree(plan->w_scale);
  delete plan;
  return ok();
}

}  // extern "C"
