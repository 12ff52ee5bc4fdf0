// Rotary positions with several axes: pair i of a head turns by position *
// inv_freq[i], the position being the one of the pair's axis.
//
// The turn is formed in fixed point: turn_i = frac(inv_freq[i] / 2 pi) in
// units of 2^-64 of a full turn, and position * turn_i modulo 2^64 keeps the
// fraction of a turn exactly, for any int32 position, where an fp32 product
// would lose a bit of the angle with every doubling of the position.  The
// upper 32 bits are split into the nearest quarter turn and a remainder of at
// most an eighth, whose sine and cosine are Taylor sums (next terms below
// 2e-9).
//
// Bytes bound it: every element is read and written once.  A thread forms the
// sines and cosines of its pairs once and walks a few heads with them.
// Measured: 2 x 25088 tokens, 16 heads of 128 bf16 (411 MB) 78 us, 5.3 TB/s, what
// a large copy reaches; 32 single tokens 4 us on the device, 7.2 a call.  Halves
// whose pairs are no whole vectors go a channel at a time: 2 x 12544 tokens, 16
// heads of 80 bf16 with 24 pairs 34 us, with 20 48.5.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "elem.h"

struct nhip_rotary_plan {
  int32_t head_dim, axes, pairs, neighbours;
  uint2* turn = nullptr;    // [pairs] low and high word of the turn
  int32_t* axis = nullptr;  // [pairs], behind the turns in one allocation
};

namespace nhip {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxAxes = 4;

struct RotaryArgs {
  const void* x;
  void* y;
  const int32_t* positions;
  const uint2* turn;
  const int32_t* axis;
  int64_t xs[3], ys[3];  // batch, token, head
  int64_t positions_stride;
  int64_t items;         // batch * tokens * parts * cols
  int32_t tokens, heads, axes, pairs, head_dim;
  int32_t cols;          // vectors of a head: rotated ones, then copied ones
  int32_t rotated;       // of them rotated
  int32_t parts, part;   // heads are walked in `parts` parts of `part`
  int32_t inverse;
};

// sine and cosine of `phase` / 2^32 turns
__device__ __forceinline__ void turn_sincos(uint32_t phase, float& s, float& c) {
  const uint32_t quarter = (phase + 0x20000000u) >> 30;
  const float t = (float)(int32_t)(phase - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float u = t * t;
  const float si = t * fmaf(u, fmaf(u, fmaf(u, fmaf(u, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -0.16666667f), 1.f);
  const float co = fmaf(u, fmaf(u, fmaf(u, fmaf(u, fmaf(u, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
  const float a = quarter & 1 ? co : si, b = quarter & 1 ? si : co;
  s = quarter & 2 ? -a : a;
  c = (quarter + 1) & 2 ? -b : b;
}

// x a + y b, rounded the same way in every form of the kernel: a token's result
// does not depend on the tensor it came with.
__device__ __forceinline__ float turned(float x, float a, float y, float b) {
#pragma clang fp contract(off)
  const float yb = y * b;
  return __builtin_fmaf(x, a, yb);
}

// One thread: V channels (and, paired as halves, the V they pair with) of one
// token, for a part of its heads.
template <class T, int V, bool NEIGHBOURS, bool STREAM>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a) {
  const int64_t item = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (item >= a.items) return;
  const int col = (int)(item % a.cols);
  const int64_t rest = item / a.cols, token = rest / a.parts;
  const int h0 = (int)(rest % a.parts) * a.part, h1 = min(h0 + a.part, a.heads);
  const int b = (int)(token / a.tokens), t = (int)(token % a.tokens);
  const T* x = (const T*)a.x + b * a.xs[0] + t * a.xs[1];
  T* y = (T*)a.y + b * a.ys[0] + t * a.ys[1];
  if (col >= a.rotated) {  // channels past the rotated ones
    const int c = 2 * a.pairs + (col - a.rotated) * V;
    for (int h = h0; h < h1; ++h) {
      float v[V];
      Vec<T, V>::load(x + h * a.xs[2] + c, v);
      Vec<T, V>::template store<STREAM>(y + h * a.ys[2] + c, v);
    }
    return;
  }
  // neighbours: V channels are V/2 pairs (a single channel never comes here
  // alone: V == 1 takes two); halves: V pairs
  constexpr int P = NEIGHBOURS ? (V > 1 ? V / 2 : 1) : V;
  const int pair = col * P;
  const int32_t* pos = a.positions + b * a.positions_stride + (int64_t)t * a.axes;
  float sn[P], cs[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const uint2 f = a.turn[pair + i];
    const int32_t p = pos[a.axis[pair + i]];
    const uint32_t up = (uint32_t)p;
    // bits 32..63 of p * turn modulo 2^64, p sign-extended
    const uint32_t phase = up * f.y + __umulhi(up, f.x) - (p < 0 ? f.x : 0u);
    turn_sincos(phase, sn[i], cs[i]);
    if (a.inverse) sn[i] = -sn[i];
  }
  if (NEIGHBOURS) {
    constexpr int W = 2 * P;
#pragma unroll 2
    for (int h = h0; h < h1; ++h) {
      const T* xh = x + h * a.xs[2] + 2 * pair;
      T* yh = y + h * a.ys[2] + 2 * pair;
      float v[W], o[W];
      if (V > 1) {
        Vec<T, W>::load(xh, v);
      } else {
        v[0] = (float)xh[0];
        v[1] = (float)xh[1];
      }
#pragma unroll
      for (int i = 0; i < P; ++i) {
        o[2 * i] = turned(v[2 * i], cs[i], v[2 * i + 1], -sn[i]);
        o[2 * i + 1] = turned(v[2 * i], sn[i], v[2 * i + 1], cs[i]);
      }
      if (V > 1) {
        Vec<T, W>::template store<STREAM>(yh, o);
      } else {
        yh[0] = (T)o[0];
        yh[1] = (T)o[1];
      }
    }
  } else {
#pragma unroll 2
    for (int h = h0; h < h1; ++h) {
      const T* xh = x + h * a.xs[2] + pair;
      T* yh = y + h * a.ys[2] + pair;
      float u[V], v[V], o[V], q[V];
      Vec<T, V>::load(xh, u);
      Vec<T, V>::load(xh + a.pairs, v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        o[i] = turned(u[i], cs[i], v[i], -sn[i]);
        q[i] = turned(u[i], sn[i], v[i], cs[i]);
      }
      Vec<T, V>::template store<STREAM>(yh, o);
      Vec<T, V>::template store<STREAM>(yh + a.pairs, q);
    }
  }
}

template <class T, int V>
int rotary_launch(RotaryArgs a, bool neighbours, int64_t tokens, hipStream_t s) {
  a.rotated = neighbours ? (V > 1 ? 2 * a.pairs / V : a.pairs) : a.pairs / V;
  a.cols = a.rotated + (a.head_dim - 2 * a.pairs) / V;
  // the sines of a thread's pairs serve up to eight heads, fewer where the
  // launch would not give every CU eight workgroups
  const int64_t want = (int64_t)8 * cu_count() * kThreads;
  a.part = (int)std::max<int64_t>(1, std::min<int64_t>({8, a.heads, tokens * a.cols * a.heads / want}));
  a.parts = (int)ceil_div(a.heads, a.part);
  a.items = tokens * a.parts * a.cols;
  const int64_t wgs = ceil_div(a.items, kThreads);
  if (wgs > 0x7fffffff) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "rotary: tensor too large");
  // us without / with: 205 MB 80.6 / 78.1, 103 MB 44.8 / 42.2, 26 MB 15.8 / 14.6
  const bool stream = V > 1 && tokens * a.heads * a.head_dim * (int64_t)sizeof(T) > kStreamBytes;
  const auto launch = [&](auto kernel) {
    NHIP_LAUNCH("rotary", kernel, dim3((uint32_t)wgs), dim3(kThreads), 0, s, a);
  };
  if (neighbours)
    stream ? launch(rotary_kernel<T, V, true, V != 1>) : launch(rotary_kernel<T, V, true, false>);
  else
    stream ? launch(rotary_kernel<T, V, false, V != 1>) : launch(rotary_kernel<T, V, false, false>);
  return check_launch("rotary");
}

template <class T>
int rotary_run(const RotaryArgs& a, bool neighbours, int64_t tokens, hipStream_t s) {
  constexpr int V = kVec<T>;
  bool vec = aligned_to(a.x, 16) && aligned_to(a.y, 16) && a.head_dim % V == 0 &&
             (neighbours ? 2 * a.pairs : a.pairs) % V == 0;
  for (int i = 0; i < 3; ++i) vec = vec && a.xs[i] % V == 0 && a.ys[i] % V == 0;
  return vec ? rotary_launch<T, V>(a, neighbours, tokens, s) : rotary_launch<T, 1>(a, neighbours, tokens, s);
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int nhip_rotary_create(int32_t head_dim, int32_t axes, const int32_t* sections, const float* inv_freq,
                       int32_t neighbours, nhip_rotary_t* plan) {
  if (!plan) return fail(NHIP_STATUS_NULL_POINTER, "rotary: null plan pointer");
  *plan = nullptr;
  if (!sections || !inv_freq) return fail(NHIP_STATUS_NULL_POINTER, "rotary: null pointer");
  if (axes < 1 || axes > kMaxAxes) return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: 1 to 4 axes");
  if (head_dim <= 0) return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: head_dim has to be positive");
  int64_t pairs = 0;
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: a section is negative");
    pairs += sections[a];
  }
  if (pairs < 1 || 2 * pairs > head_dim)
    return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: the sections have to hold 1 to head_dim / 2 pairs");
  uint2* dev = nullptr;
  try {
    // turns, then axes
    std::vector<uint32_t> host(3 * (size_t)pairs);
    for (int64_t i = 0; i < pairs; ++i) {
      if (!std::isfinite(inv_freq[i])) return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "rotary: inv_freq has to be finite");
      // x87 long double: 64 bits of fraction, what a turn has
      const long double turns = (long double)inv_freq[i] / 6.283185307179586476925286766559L;
      const long double frac = turns - std::floor(turns);
      const long double scaled = std::floor(frac * 18446744073709551616.0L + 0.5L);
      const uint64_t f = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
      host[2 * i] = (uint32_t)f;
      host[2 * i + 1] = (uint32_t)(f >> 32);
    }
    for (int64_t i = 0, a = 0, end = sections[0]; i < pairs; ++i) {
      while (i >= end) end += sections[++a];
      host[2 * pairs + i] = (uint32_t)a;
    }
    NHIP_TRY(check_hip(hipMalloc(reinterpret_cast<void**>(&dev), host.size() * 4), "hipMalloc(rotary)"));
    const int st = check_hip(hipMemcpy(dev, host.data(), host.size() * 4, hipMemcpyHostToDevice), "hipMemcpy(rotary)");
    if (st != NHIP_STATUS_SUCCESS) {
      (void)hipFree(dev);
      return st;
    }
    nhip_rotary_plan* p = new nhip_rotary_plan;
    p->head_dim = head_dim;
    p->axes = axes;
    p->pairs = (int32_t)pairs;
    p->neighbours = neighbours != 0;
    p->turn = dev;
    p->axis = (int32_t*)(dev + pairs);
    *plan = p;
  } catch (const std::bad_alloc&) {
    (void)hipFree(dev);
    return fail(NHIP_STATUS_DEVICE_ERROR, "rotary: out of host memory");
  }
  return ok();
}

int nhip_rotary_forward(nhip_rotary_t plan, const void* x, int32_t dtype, int32_t batch, int32_t tokens, int32_t heads,
                        const int64_t* x_strides, const int32_t* positions, int64_t positions_stride, int32_t inverse,
                        void* y, const int64_t* y_strides, void* stream) {
  if (!plan || !x_strides || !y_strides) return fail(NHIP_STATUS_NULL_POINTER, "rotary: null pointer");
  const int es = elem_size(dtype);
  if (!es) return fail(NHIP_STATUS_UNSUPPORTED, "rotary: dtype has to be F32, F16 or BF16");
  if (batch < 0 || tokens < 0 || heads < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: negative extent");
  if (batch == 0 || tokens == 0 || heads == 0) return ok();
  if (!x || !y || !positions) return fail(NHIP_STATUS_NULL_POINTER, "rotary: null pointer");
  if (!aligned_to(x, es) || !aligned_to(y, es) || !aligned_to(positions, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "rotary: a tensor is not aligned to its type");
  RotaryArgs a{};
  a.x = x;
  a.y = y;
  a.positions = positions;
  a.turn = plan->turn;
  a.axis = plan->axis;
  for (int i = 0; i < 3; ++i) {
    if (x_strides[i] < 0 || y_strides[i] < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: negative stride");
    a.xs[i] = x_strides[i];
    a.ys[i] = y_strides[i];
  }
  if ((batch > 1 && !a.ys[0]) || (tokens > 1 && !a.ys[1]) || (heads > 1 && a.ys[2] < plan->head_dim))
    return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: rows of the output overlap");
  if (positions_stride < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "rotary: negative stride");
  a.positions_stride = positions_stride;
  a.tokens = tokens;
  a.heads = heads;
  a.axes = plan->axes;
  a.pairs = plan->pairs;
  a.head_dim = plan->head_dim;
  a.inverse = inverse;
  const int64_t total = (int64_t)batch * tokens;
  if (total > (int64_t(1) << 42) / heads / plan->head_dim)
    return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "rotary: tensor too large");
  return NHIP_FOR_ELEM(dtype, T, rotary_run<T>(a, plan->neighbours, total, as_stream(stream)));
}

int nhip_rotary_destroy(nhip_rotary_t plan) {
  if (!plan) return ok();
  (void)hipFree(plan->turn);
  delete plan;
  return ok();
}

}  // extern "C"
