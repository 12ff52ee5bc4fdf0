// Group norm with an activation into channels-last tokens:
//   y = act((x - mean_g) / sqrt(var_g + eps) * gamma_c + beta_c).
//
// Bytes bound it.  Where a few groups of an image fit a workgroup's registers,
// it reads them once, sums, and writes y.  Else two launches: the statistics of
// every (image, group) over chunks of pixels (a mean and a sum of squared
// deviations each), and a pass that merges them and writes y: x is read twice,
// the second time from the last-level cache where the tensor fits.
// Measured: 32 x 3136 x 256 bf16 26.2-26.8 us a call (103 MB moved, 3.9 TB/s; two
// launches 33), 128 x 784 x 512 bf16 39.6 us (5.2 TB/s, as a large copy; two
// launches 56); 8 x 50175 x 320 f16, in two launches, 135-142 us (some 48 and 83-94;
// floor with one reading 99).  Images two at a time, so that the second
// reading stays in the last-level cache, were no faster (153).  Small tensors
// take one launch that reads twice (5.5 us on the device at 1 x 128 x 28 x 28
// fp32 blobs; a call is bound by the host's 7.1).
//
// Statistics: sums of x - s and (x - s)^2 in 64 bits, s being one of the values
// (16-bit types: blocks of at most kBlock values in fp32 first); means and
// squared deviations of channels and chunks are then merged in 64 bits (the sum
// of squares about a common mean is the sum of the parts' plus count *
// (difference of means)^2).  A large mean beside a small spread loses nothing so,
// as it would in E[x^2] - E[x]^2, nor does an s far from all others: what the
// subtraction leaves is at least 1 / (count + 1) of the sum.  (Thread sums of
// fp32 were off by up to 1e-3 there.)
#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "elem.h"

struct nhip_norm_plan {
  int32_t channels, groups, act;
  float eps;
  float* affine = nullptr;  // gamma [channels], beta [channels]
};

namespace nhip {
namespace {

constexpr int kThreads = 512;      // of a workgroup, tokens
constexpr int kBlobThreads = 256;  // blobs, two launches
constexpr int kOneThreads = 512;   // of a workgroup that does its groups alone
constexpr int kHeld = 16;  // vectors that a thread holds at most (single reading)
constexpr int kMaxChannels = 4096;
constexpr int kMaxChunks = 256;  // parts of an image: what each workgroup of the second pass merges
constexpr int kDeep = 4;         // vectors of a thread under way at once
constexpr int kTile = 64;        // pixels and channels of a transposed tile (blobs)

struct NormArgs {
  const void* x;
  void* y;
  double2* part;  // [n][chunks][groups]: mean, sum of squared deviations
  const float* affine;
  int64_t pixels, image_stride, row_stride;
  int channels, groups, cpg, act;
  int chunks;           // of an image; 0: one launch
  int64_t chunk;        // pixels of a chunk (the last may have fewer)
  float eps;
};

template <int ACT>
__device__ __forceinline__ float activate(float y) {
  if (ACT == NHIP_ACT_RELU) return y < 0.f ? 0.f : y;  // NaN stays
  if (ACT == NHIP_ACT_SILU) return y * __builtin_amdgcn_rcpf(1.f + __expf(-y));
  return y;
}

// Lanes of a wave that share one group: a power of two, so that their sums
// are butterflies inside the wave.
template <int TH>
__device__ __forceinline__ int team_of(int groups) {
  int t = 64;
  while (t > 1 && (TH / t) < groups) t >>= 1;
  return t;
}
template <class S>
__device__ __forceinline__ S team_sum(S v, int team) {
  for (int o = team >> 1; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// First and second powers that a thread adds up.  WIDE: each value, taken from
// `shift`, in 64 bits.
template <class T, bool WIDE>
struct Powers {
  double s1 = 0.0, s2 = 0.0;
  __device__ __forceinline__ void begin(float) {}
  __device__ __forceinline__ void add(float x, float shift) {
    const double d = (double)x - (double)shift;
    s1 += d;
    s2 = fma(d, d, s2);
  }
  __device__ __forceinline__ void end(int) {}
  __device__ __forceinline__ double first() const { return s1; }
  __device__ __forceinline__ double second() const { return s2; }
};
// Else (16-bit types): a block of at most kBlock values in fp32, and the blocks
// in 64 bits (a value's conversion to 64 bits takes four instructions' time).
// Sums of so few values of 11 bits or less are nearly always exact.  So are those
// of bf16 squares, 16 bits each, unless values differ by factors, and then the
// mean's square takes little from them.  fp16's squares are taken from the mean
// of a few of the block's values, which is near the others or, beside a value far
// off, at most a fourth as far.  us with 64 bits value by value / in blocks: 32 x
// 160 x 50176 f16 blobs 537 / 484, 64 x 3136 x 256 bf16 tokens 56.3 / 53.2.
constexpr int kBlock = 32;
template <class T>
struct Block {
  static constexpr bool centred = std::is_same<T, f16>::value;
  float from, b1, b2;
  int n;
  __device__ __forceinline__ void begin(float x, int values) {
    from = x;
    b1 = b2 = 0.f;
    n = values;
  }
  __device__ __forceinline__ void add(float x, float) {
    const float d = centred ? x - from : x;
    b1 += x;
    b2 = fmaf(d, d, b2);
  }
  // sums of x and x^2
  __device__ __forceinline__ double first() const { return b1; }
  __device__ __forceinline__ double second() const {
    if (!centred) return b2;
    const double c = from, u = b1;
    return fma(c, fma((double)-n, c, u + u), (double)b2);
  }
};
template <class T>
struct Powers<T, false> {
  double s1 = 0.0, s2 = 0.0;
  Block<T> block;
  __device__ __forceinline__ void begin(float x) { block.begin(x, 0); }
  __device__ __forceinline__ void add(float x, float) { block.add(x, 0.f); }
  __device__ __forceinline__ void end(int n) {
    block.n = n;
    s1 += block.first();
    s2 += block.second();
  }
  __device__ __forceinline__ double first() const { return s1; }
  __device__ __forceinline__ double second() const { return s2; }
};

// Mean and squared deviations of `count` values from their sums (WIDE: those of
// x - shift).  Rounding may leave the latter below 0; NaN, of values that are
// not all finite, stays.
template <bool WIDE>
__device__ __forceinline__ double2 moments(double s1, double s2, double shift, double count) {
  if (!WIDE) {
    s2 = fma(count * shift, shift, fma(-2.0 * shift, s1, s2));
    s1 = fma(-count, shift, s1);
  }
  const double d = s1 / count, v = fma(-s1, d, s2);
  return make_double2(shift + d, v < 0.0 ? 0.0 : v);
}
// Whether fp32 may have lost squares: above its range, or below it where eps
// does not hide that.  Then the sums are formed again, WIDE.
__device__ __forceinline__ bool out_of_range(double2 m, double count, float eps) {
  return !(m.y <= 1.7976931348623157e308) || (eps < 0x1p-110f && m.y < count * 0x1p-110);
}

// Merges the chunks of image `n` for groups [g0, g1): mean and 1/sqrt(var + eps)
// to stat[g - g0].
template <int TH>
__device__ void merge_chunks(const NormArgs& a, int n, int g0, int g1, float2* stat) {
  const int team = team_of<TH>(g1 - g0), lane = threadIdx.x & (team - 1);
  const double2* part = a.part + (int64_t)n * a.chunks * a.groups;
  const double last = (double)(a.pixels - (int64_t)(a.chunks - 1) * a.chunk), total = (double)a.pixels;
  for (int gb = g0; gb < g1; gb += TH / team) {  // uniform: all lanes of a team stay in the butterflies
    const int g = gb + threadIdx.x / team;
    const bool in = g < g1;
    double m = 0.0;
    for (int k = lane; in && k < a.chunks; k += team)
      m += part[(int64_t)k * a.groups + g].x * (k == a.chunks - 1 ? last : (double)a.chunk);
    m = team_sum(m, team) / total;
    double v = 0.0;
    for (int k = lane; in && k < a.chunks; k += team) {
      const double2 p = part[(int64_t)k * a.groups + g];
      const double d = p.x - m;
      v += p.y + (k == a.chunks - 1 ? last : (double)a.chunk) * a.cpg * d * d;
    }
    v = team_sum(v, team) / (total * a.cpg);
    if (in && lane == 0) stat[g - g0] = make_float2((float)m, (float)(1.0 / sqrt(v + (double)a.eps)));
  }
}

// LDS that sum_channels takes, in values of 64 bits.
__host__ __device__ constexpr int sums_place(int v, int threads) { return v * (threads + 64 / v) + 2 * threads + 1; }

// Adds the sums of `rows` threads for each of `cols` vectors of channels
// (thread row * cols + col), those of a channel by as many threads as there are
// for it, then by one: means and squared deviations of `count` values each to
// ch.  shift: what each channel's values are taken from.  First and second powers
// go through the same place (red, sums_place) one after the other, a vector's
// channels in rows of their own, which begin in different banks.  Whether some
// channel is out_of_range.
template <bool WIDE, class T, int V, int TH, class P>
__device__ bool sum_channels(const NormArgs& a, const T* shift, int cols, int rows, int col, int row, double count,
                             double2* ch, double* red, const P (&sums)[V]) {
  constexpr int ROW = TH + 64 / V;
  double* more = red + V * ROW;
  int* found = reinterpret_cast<int*>(more + 2 * TH);
  const int mine = threadIdx.x, cv = cols * V;
  const int parts = rows / V;  // threads of a channel; 0: a thread has several channels
  const float from = row < V && row < rows ? (float)shift[col * V + row] : 0.f;
  bool odd = false;
  const auto done = [&](int c, double u1, double u2, float s) {
    ch[c] = moments<WIDE>(u1, u2, (double)s, count);
    odd |= out_of_range(ch[c], count, a.eps);
  };
  const auto put = [&](int power) {
    __syncthreads();
    if (power == 1 && mine == 0) *found = 0;  // (all have read what an earlier call left)
    if (row < rows)
#pragma unroll
      for (int i = 0; i < V; ++i) red[i * ROW + mine] = power == 1 ? sums[i].first() : sums[i].second();
    __syncthreads();
  };
  const auto add = [&](int i, int part, int step) {  // rows part, part + step, ..
    const double* of = red + i * ROW + col;
    double u = 0.0;
#pragma unroll 4
    for (int r = part; r < rows; r += step) u += of[r * cols];
    return u;
  };
  if (parts) {  // uniform
    put(1);
    const bool in = row < parts * V;
    const double u1 = in ? add(row % V, row / V, parts) : 0.0;
    put(2);
    const double u2 = in ? add(row % V, row / V, parts) : 0.0;
    if (in) {  // vectors' i-th channels side by side, as the threads of row i
      const int to = row / V * cv + row % V * cols + col;
      more[to] = u1;
      more[TH + to] = u2;
    }
    __syncthreads();
    if (row < V) {
      double v1 = 0.0, v2 = 0.0;
#pragma unroll 8
      for (int q = 0; q < parts; ++q) {
        v1 += more[q * cv + mine];
        v2 += more[TH + q * cv + mine];
      }
      done(col * V + row, v1, v2, from);
    }
  } else {
    put(1);
    if (row < rows)
      for (int i = row; i < V; i += rows) ch[col * V + i].x = add(i, 0, 1);
    put(2);
    if (row < rows)
      for (int i = row; i < V; i += rows) {
        const int c = col * V + i;
        done(c, ch[c].x, add(i, 0, 1), (float)shift[c]);
      }
  }
  if (!WIDE && odd) *found = 1;
  __syncthreads();
  return !WIDE && *found;
}

// Means and squared deviations of channels [c0, c0 + cn) over pixels [p0, p1)
// of one image (x: its first pixel), channels last, to ch[0, cn).  A thread
// keeps its V channels and walks pixels; `red` holds the threads' sums.
// Whether some channel is out_of_range.
template <bool WIDE, class T, int V, int TH>
__device__ bool channel_powers(const NormArgs& a, const T* x, int c0, int cn, int64_t p0, int64_t p1, double2* ch, double* red) {
  bool odd = false;
  const int vecs = cn / V;
  for (int v0 = 0; v0 < vecs; v0 += TH) {
    const int cols = min(TH, vecs - v0), rows = TH / cols;
    const int col = threadIdx.x % cols, row = threadIdx.x / cols;
    Powers<T, WIDE> sums[V];
    if (row < rows) {
      const T* px = x + c0 + (int64_t)(v0 + col) * V;
      float shift[V];
      if constexpr (WIDE) Vec<T, V>::load(px + p0 * a.row_stride, shift);
      int n = 0;  // values of the open block
      const auto add = [&](const float(&t)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) sums[i].add(t[i], WIDE ? shift[i] : 0.f);
      };
      const auto end = [&] {
#pragma unroll
        for (int i = 0; i < V; ++i) sums[i].end(n);
        n = 0;
      };
      const int64_t step = rows * a.row_stride;
      int64_t p = p0 + row;
      const T* at = px + p * a.row_stride;
      for (; p + (kDeep - 1) * rows < p1; p += kDeep * rows, at += kDeep * step) {
        float t[kDeep][V];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) Vec<T, V>::load(at + u * step, t[u]);
        if (n == 0)
#pragma unroll
          for (int i = 0; i < V; ++i) sums[i].begin((t[0][i] + t[1][i] + t[2][i] + t[3][i]) * 0.25f);
#pragma unroll
        for (int u = 0; u < kDeep; ++u) add(t[u]);
        n += kDeep;
        if (n > kBlock - kDeep) end();
      }
      for (; p < p1; p += rows, at += step) {  // fewer than kDeep of them, for which the block has room
        float t[V];
        Vec<T, V>::load(at, t);
        if (n == 0)
#pragma unroll
          for (int i = 0; i < V; ++i) sums[i].begin(t[i]);
        add(t);
        ++n;
      }
      if (n) end();
    }
    odd |= sum_channels<WIDE, T, V, TH>(a, x + p0 * a.row_stride + c0 + v0 * V, cols, rows, col, row, (double)(p1 - p0), ch + v0 * V, red, sums);
  }
  return odd;
}
static_assert(kDeep == 4, "the mean of a block's first values");

template <class T, int V, int TH>
__device__ __forceinline__ void channel_moments(const NormArgs& a, const T* x, int c0, int cn, int64_t p0, int64_t p1, double2* ch, double* red) {
  if constexpr (sizeof(T) == 4)
    channel_powers<true, T, V, TH>(a, x, c0, cn, p0, p1, ch, red);
  else if (__builtin_expect(channel_powers<false, T, V, TH>(a, x, c0, cn, p0, p1, ch, red), false))
    channel_powers<true, T, 1, TH>(a, x, c0, cn, p0, p1, ch, red);  // (V = 1: few registers)
}

// Merges channels of `count` values each into `groups` groups: calls
// done(group, mean, squared deviations) in one lane for each.
template <int TH, class F>
__device__ __forceinline__ void merge_channels(const NormArgs& a, const double2* ch, int groups, double count, F done) {
  const int team = team_of<TH>(groups), lane = threadIdx.x & (team - 1);
  for (int gb = 0; gb < groups; gb += TH / team) {
    const int g = gb + threadIdx.x / team;
    const bool in = g < groups;
    const double2* of = ch + g * a.cpg;
    double m = 0.0;
    for (int c = lane; in && c < a.cpg; c += team) m += of[c].x;
    m = team_sum(m, team) / a.cpg;
    double v = 0.0;
    for (int c = lane; in && c < a.cpg; c += team) {
      const double d = of[c].x - m;
      v += of[c].y + count * d * d;
    }
    v = team_sum(v, team);
    if (in && lane == 0) done(g, m, v);
  }
}

// y of channels [c0, c0 + cn) over pixels [p0, p1), channels last; stat: of
// the groups from the one that c0 begins.
template <class T, int V, int ACT, int TH, bool STREAM>
__device__ void apply_tokens(const NormArgs& a, const T* x, T* y, int c0, int cn, int64_t p0, int64_t p1, const float2* stat) {
  const int vecs = cn / V;
  for (int v0 = 0; v0 < vecs; v0 += TH) {
    const int cols = min(TH, vecs - v0), rows = TH / cols;
    const int col = threadIdx.x % cols, row = threadIdx.x / cols;
    if (row >= rows) continue;
    const int c = (v0 + col) * V;
    float mean[V], scale[V], beta[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 s = stat[(c + i) / a.cpg];
      mean[i] = s.x;
      scale[i] = s.y * a.affine[c0 + c + i];
      beta[i] = a.affine[a.channels + c0 + c + i];
    }
    const auto result = [&](float(&t)[V]) {
#pragma unroll
      for (int i = 0; i < V; ++i) t[i] = activate<ACT>(fmaf(t[i] - mean[i], scale[i], beta[i]));
    };
    const int64_t in = rows * a.row_stride, out = (int64_t)rows * a.channels;
    int64_t p = p0 + row;
    const T* from = x + p * a.row_stride + c0 + c;
    T* to = y + p * a.channels + c0 + c;
    for (; p + (kDeep - 1) * rows < p1; p += kDeep * rows, from += kDeep * in, to += kDeep * out) {
      float t[kDeep][V];
#pragma unroll
      for (int u = 0; u < kDeep; ++u) Vec<T, V>::load(from + u * in, t[u]);
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        result(t[u]);
        Vec<T, V>::template store<STREAM>(to + u * out, t[u]);
      }
    }
    for (; p < p1; p += rows, from += in, to += out) {
      float t[V];
      Vec<T, V>::load(from, t);
      result(t);
      Vec<T, V>::template store<STREAM>(to, t);
    }
  }
}

// Statistics of one chunk of one image, channels last.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void norm_stats_tokens_kernel(NormArgs a) {
  extern __shared__ double2 lds[];  // [channels] mean, deviations; then the threads' sums
  const int n = blockIdx.x / a.chunks, k = blockIdx.x % a.chunks;
  const int64_t p0 = (int64_t)k * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
  channel_moments<T, V, kThreads>(a, (const T*)a.x + n * a.image_stride, 0, a.channels, p0, p1, lds, (double*)(lds + a.channels));
  merge_channels<kThreads>(a, lds, a.groups, (double)(p1 - p0),
                 [&](int g, double m, double v) { a.part[(int64_t)blockIdx.x * a.groups + g] = make_double2(m, v); });
}

// Result of `each` groups over `run` chunks of pixels.
template <class T, int V, int ACT, bool STREAM>
__global__ __launch_bounds__(kThreads) void norm_apply_tokens_kernel(NormArgs a, int each, int run, int runs) {
  extern __shared__ float2 stats[];  // [each]
  const int k = blockIdx.x % runs, rest = blockIdx.x / runs;
  const int g0 = rest % (a.groups / each) * each, n = rest / (a.groups / each);
  merge_chunks<kThreads>(a, n, g0, g0 + each, stats);
  __syncthreads();
  const int64_t p0 = (int64_t)k * run * a.chunk, p1 = min(p0 + run * a.chunk, a.pixels);
  apply_tokens<T, V, ACT, kThreads, STREAM>(a, (const T*)a.x + n * a.image_stride, (T*)a.y + n * a.pixels * a.channels,
                                    g0 * a.cpg, each * a.cpg, p0, p1, stats);
}

// Small images in one launch: a workgroup does a few whole groups of an
// image, statistics and result.
template <class T, int V, int ACT>
__global__ __launch_bounds__(kOneThreads) void norm_one_tokens_kernel(NormArgs a, int groups) {
  extern __shared__ double2 lds[];  // [channels of the groups]; then the threads' sums, and in their place the statistics
  const int parts = a.groups / groups, n = blockIdx.x / parts, g0 = blockIdx.x % parts * groups;
  const T* x = (const T*)a.x + n * a.image_stride;
  const int cn = groups * a.cpg;
  channel_moments<T, V, kOneThreads>(a, x, g0 * a.cpg, cn, 0, a.pixels, lds, (double*)(lds + cn));
  float2* stats = reinterpret_cast<float2*>(lds + cn);
  const double all = (double)a.pixels * a.cpg, eps = a.eps;
  merge_channels<kOneThreads>(a, lds, groups, (double)a.pixels,
                 [&](int g, double m, double v) { stats[g] = make_float2((float)m, (float)(1.0 / sqrt(v / all + eps))); });
  __syncthreads();
  apply_tokens<T, V, ACT, kOneThreads, false>(a, x, (T*)a.y + n * a.pixels * a.channels, g0 * a.cpg, cn, 0, a.pixels, stats);
}

// A workgroup does a few whole groups of an image whose values its threads
// hold, so that x is read once: all loads first, then the statistics, then the
// results.  (At most kHeld times the workgroup's rows of pixels; whole vectors.)
template <class T, int V, int ACT, int TH, bool STREAM>
__global__ __launch_bounds__(TH, 4) void norm_held_tokens_kernel(NormArgs a, int groups, int wgs) {
  extern __shared__ double2 lds[];  // as norm_one_tokens_kernel's
  // workgroups go to the eight dies in turn: an image's parts, which share
  // lines of memory, to one of them
  const int wg = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (wg >= wgs) return;
  const int parts = a.groups / groups, n = wg / parts, c0 = wg % parts * groups * a.cpg;
  const int cn = groups * a.cpg, cols = cn / V, rows = TH / cols, pixels = (int)a.pixels;
  const int col = threadIdx.x % cols, row = threadIdx.x / cols;
  const T* x = (const T*)a.x + n * a.image_stride + c0;
  typename Vec<T, V>::type held[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u)  // (past the last pixel: that one again)
    if (u * rows < pixels) held[u] = *reinterpret_cast<const typename Vec<T, V>::type*>(x + min(row + u * rows, pixels - 1) * a.row_stride + col * V);
  float shift[V];
  if constexpr (sizeof(T) == 4) Vec<T, V>::load(x + col * V, shift);
  const int mine = row < rows ? (pixels - row + rows - 1) / rows : 0;  // vectors that count
  constexpr bool WIDE = sizeof(T) == 4;
  static_assert(kHeld <= kBlock, "one block");
  bool odd;
  {
    typename std::conditional<WIDE, Powers<T, WIDE>, Block<T>>::type sums[V];
    if constexpr (!WIDE) {
      const float part = 1.f / (float)max(1, min(mine, 4));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float from = (float)held[0][i];
#pragma unroll
        for (int u = 1; u < 4; ++u) from += u < mine ? (float)held[u][i] : 0.f;
        sums[i].begin(from * part, mine);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) asm volatile("" : "+v"(held[u]));  // widened again below, not kept
    }
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (u < mine)
#pragma unroll
        for (int i = 0; i < V; ++i) sums[i].add((float)held[u][i], WIDE ? shift[i] : 0.f);
    odd = sum_channels<WIDE, T, V, TH>(a, x, cols, rows, col, row, (double)a.pixels, lds, (double*)(lds + cn), sums);
  }
  if (__builtin_expect(odd, false)) channel_powers<true, T, 1, TH>(a, x, 0, cn, 0, a.pixels, lds, (double*)(lds + cn));
  float2* stats = reinterpret_cast<float2*>(lds + cn);
  const double all = (double)a.pixels * a.cpg, eps = a.eps;
  merge_channels<TH>(a, lds, groups, (double)a.pixels,
                 [&](int g, double m, double v) { stats[g] = make_float2((float)m, (float)(1.0 / sqrt(v / all + eps))); });
  __syncthreads();
  float mean[V], scale[V], beta[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float2 s = stats[(col * V + i) / a.cpg];
    mean[i] = s.x;
    scale[i] = s.y * a.affine[c0 + col * V + i];
    beta[i] = a.affine[a.channels + c0 + col * V + i];
  }
  T* y = (T*)a.y + (n * a.pixels + row) * a.channels + c0 + col * V;
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u < mine) {
      float t[V];
#pragma unroll
      for (int i = 0; i < V; ++i) t[i] = activate<ACT>(fmaf((float)held[u][i] - mean[i], scale[i], beta[i]));
      Vec<T, V>::template store<STREAM>(y + (int64_t)u * rows * a.channels, t);
    }
}

// Mean and squared deviations of pixels [p0, p1) of one group's channels,
// channels first (x: the group's first channel), the same in every thread.
template <class T, int V, int TH>
__device__ double2 group_moments(const NormArgs& a, const T* x, int64_t p0, int64_t p1) {
  __shared__ double red1[TH / 64], red2[TH / 64];
  const float shift = (float)x[p0];
  const int vecs = (int)((p1 - p0) / V);
  const int lanes = min(TH, (vecs + 63) / 64 * 64);
  const int rows = TH / lanes, row = threadIdx.x / lanes, col = threadIdx.x % lanes;
  const double count = (double)(p1 - p0) * a.cpg;
  const auto pass = [&](auto wide) {
    Powers<T, wide> sums;
    const auto add = [&](auto& t, int n) {  // n vectors, a block
      sums.begin(n > 1 ? (t[0][0] + t[n / 4][0] + t[n / 2][0] + t[n - 1][0]) * 0.25f
                       : (t[0][0] + t[0][V / 4] + t[0][V / 2] + t[0][V - 1]) * 0.25f);
      for (int u = 0; u < n; ++u)
#pragma unroll
        for (int i = 0; i < V; ++i) sums.add(t[u][i], shift);
      sums.end(n * V);
    };
    static_assert(kDeep * V <= kBlock, "one block");
    if (row < rows)
      for (int c = row; c < a.cpg; c += rows) {
        const T* at = x + c * a.row_stride + p0;
        int v = col;
        for (; v + (kDeep - 1) * lanes < vecs; v += kDeep * lanes) {
          float t[kDeep][V];
#pragma unroll
          for (int u = 0; u < kDeep; ++u) Vec<T, V>::load(at + (int64_t)(v + u * lanes) * V, t[u]);
          add(t, kDeep);
        }
#pragma unroll 3
        for (; v < vecs; v += lanes) {
          float t[1][V];
          Vec<T, V>::load(at + (int64_t)v * V, t[0]);
          add(t, 1);
        }
      }
    const double s1 = team_sum(sums.s1, 64), s2 = team_sum(sums.s2, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      red1[threadIdx.x / 64] = s1;
      red2[threadIdx.x / 64] = s2;
    }
    __syncthreads();
    double u1 = 0.0, u2 = 0.0;
    for (int i = 0; i < TH / 64; ++i) {
      u1 += red1[i];
      u2 += red2[i];
    }
    return moments<wide>(u1, u2, (double)shift, count);
  };
  if constexpr (sizeof(T) == 4) {
    return pass(std::true_type());
  } else {
    const double2 m = pass(std::false_type());
    return out_of_range(m, count, a.eps) ? pass(std::true_type()) : m;  // the same in all threads
  }
}

// Statistics of one chunk of pixels of one group, channels first.
template <class T, int V>
__global__ __launch_bounds__(kBlobThreads) void norm_stats_blobs_kernel(NormArgs a) {
  const int g = blockIdx.x % a.groups, nk = blockIdx.x / a.groups;
  const int n = nk / a.chunks, k = nk % a.chunks;
  const int64_t p0 = (int64_t)k * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
  const double2 m = group_moments<T, V, kBlobThreads>(a, (const T*)a.x + n * a.image_stride + (int64_t)g * a.cpg * a.row_stride, p0, p1);
  if (threadIdx.x == 0) a.part[(int64_t)nk * a.groups + g] = m;
}

// Small images in one launch, channels first: a workgroup does one group of
// an image.  Lanes run along the group's channels, then pixels: results leave
// in pieces of a group's channels, values come in runs of 64 / channels pixels.
template <class T, int V, int ACT>
__global__ __launch_bounds__(kOneThreads) void norm_one_blobs_kernel(NormArgs a, FastDiv by_cpg) {
  const int g = blockIdx.x % a.groups, n = blockIdx.x / a.groups;
  const T* x = (const T*)a.x + n * a.image_stride + (int64_t)g * a.cpg * a.row_stride;
  T* y = (T*)a.y + n * a.pixels * a.channels + g * a.cpg;
  const double2 s = group_moments<T, V, kOneThreads>(a, x, 0, a.pixels);
  const float mean = (float)s.x, rstd = (float)(1.0 / sqrt(s.y / ((double)a.pixels * a.cpg) + (double)a.eps));
  const int all = (int)a.pixels * a.cpg;
  const float* gamma = a.affine + g * a.cpg;
#pragma unroll 4
  for (int i = threadIdx.x; i < all; i += kOneThreads) {
    const int p = fdiv(i, by_cpg), c = i - p * a.cpg;
    const float v = (float)x[c * a.row_stride + p];
    y[(int64_t)p * a.channels + c] = (T)activate<ACT>(fmaf(v - mean, rstd * gamma[c], gamma[a.channels + c]));
  }
}

// A tile of kTile channels x kTile pixels through LDS: read along the pixels,
// written along the channels.
template <class T, int ACT>
__global__ __launch_bounds__(kBlobThreads) void norm_apply_blobs_kernel(NormArgs a, int ptiles, int ctiles) {
  __shared__ float tile[kTile][kTile + 1];
  __shared__ float2 stat[kTile];
  const int pt = blockIdx.x % ptiles, rest = blockIdx.x / ptiles;
  const int c0 = rest % ctiles * kTile, n = rest / ctiles;
  const int64_t p0 = (int64_t)pt * kTile;
  const int cn = min(kTile, a.channels - c0), pn = (int)min((int64_t)kTile, a.pixels - p0);
  const int g0 = c0 / a.cpg, g1 = (c0 + cn - 1) / a.cpg + 1;
  merge_chunks<kBlobThreads>(a, n, g0, g1, stat);
  const T* x = (const T*)a.x + n * a.image_stride + p0;
  T* y = (T*)a.y + (n * a.pixels + p0) * a.channels + c0;
  const int lane = threadIdx.x % kTile, row = threadIdx.x / kTile;
#pragma unroll 4
  for (int c = row; c < cn; c += kBlobThreads / kTile)
    if (lane < pn) tile[c][lane] = (float)x[(int64_t)(c0 + c) * a.row_stride + lane];
  __syncthreads();
  if (lane >= cn) return;
  const float2 s = stat[(c0 + lane) / a.cpg - g0];
  const float scale = s.y * a.affine[c0 + lane], beta = a.affine[a.channels + c0 + lane];
#pragma unroll 4
  for (int p = row; p < pn; p += kBlobThreads / kTile)
    y[(int64_t)p * a.channels + lane] = (T)activate<ACT>(fmaf(tile[lane][p] - s.x, scale, beta));
}

// Groups that one workgroup of the single launch does: those whose channels
// fill 64 bytes of a pixel (tokens), one (blobs).  0: two launches.
//
// One launch spares the second's 4 us where the call is bound by launches; but
// a workgroup walks its groups' pixels alone.  Measured, us a call (two
// launches / one): tokens of 50 KB to a workgroup 12.6 / 9.9 (784 x 512 bf16)
// and 12.1 / 8.9 (fp32), of 200 KB 13.2 / 15.5 (fp32) and 15.2 / 19.4 (bf16);
// blobs of 3136 values 10.8 / 6.7, of 6272 11.1 / 8.0 (8 images 13.1 / 12.1), of 12544
// 10.9 / 11.5 (8 images 16.3 / 18.3).  Of tensors past 10 MB (tokens) or 16 MB
// (blobs) the launches no longer count: 32 x 784 x 512 fp32 31 / 43.
int groups_of_one(int channels, int groups, int layout, int es, int64_t n, int64_t pixels) {
  const int cpg = channels / groups;
  int each = 1;
  if (layout == NHIP_LAYOUT_TOKENS)
    while (each * cpg * es < 64 && groups % (2 * each) == 0) each *= 2;
  const int64_t values = pixels * each * cpg;
  const int force = setting_int("NHIP_NORM_ONE", -1);
  if (force == 0 || force == 2 || values > (1 << 28) || n * (groups / each) > 0x7fffffff) return 0;
  const int64_t bytes = n * pixels * channels * es;
  return force == 1 || (layout == NHIP_LAYOUT_TOKENS ? values * es <= 65536 && bytes <= 10000000
                                                     : values <= 8192 && bytes <= 16000000) ? each : 0;
}

// Chunks of an image: enough workgroups for two to a CU (tokens) or four
// (blobs, smaller ones), each of at least 8192 values, and few enough to be
// merged by every workgroup of the second pass.  Tokens, us a call at 2 / 3 / 4
// to a CU: 32 x 3136 x 256 bf16 32.7 / 33.7 / 34.7, 8 x 50175 x 320 f16 172 /
// 180 / 179; one image of 12544 x 320 fp32 in 128 / 256 / 512 chunks 23.6 /
// 19.8 / 25.4 (all before results past the caches and the sums in 64 bits:
// 33.3, 142 and 17.9 as chosen now).
void chunks_of(int channels, int64_t n, int64_t pixels, int per_image, NormArgs* a) {
  const int64_t want = ceil_div((int64_t)(per_image == 1 ? 2 : 4) * cu_count(), n * per_image);
  const int64_t fit = std::max<int64_t>(1, pixels * channels / per_image / 8192);
  int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({want, fit, (int64_t)kMaxChunks, pixels}));
  a->chunk = round_up(ceil_div(pixels, chunks), 8);  // whole vectors along the pixels (blobs)
  a->chunks = (int)ceil_div(pixels, a->chunk);
}

int norm_args(const nhip_norm_plan* p, int32_t dtype, int32_t layout, int32_t n, int64_t pixels, NormArgs* a, int* one) {
  if (!p) return fail(NHIP_STATUS_NULL_POINTER, "group norm: null plan");
  if (!elem_size(dtype)) return fail(NHIP_STATUS_UNSUPPORTED, "group norm: dtype has to be F32, F16 or BF16");
  if (layout != NHIP_LAYOUT_TOKENS && layout != NHIP_LAYOUT_BLOBS)
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "group norm: unknown layout");
  if (n < 0 || pixels < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "group norm: negative extent");
  if (n && pixels > (int64_t(1) << 40) / n / p->channels)
    return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "group norm: tensor too large");
  a->pixels = pixels;
  a->channels = p->channels;
  a->groups = p->groups;
  a->cpg = p->channels / p->groups;
  a->act = p->act;
  a->eps = p->eps;
  a->affine = p->affine;
  *one = n && pixels ? groups_of_one(p->channels, p->groups, layout, elem_size(dtype), n, pixels) : 0;
  if (n && pixels && !*one) {
    chunks_of(p->channels, n, pixels, layout == NHIP_LAYOUT_BLOBS ? p->groups : 1, a);
    const int64_t wgs = std::max<int64_t>((int64_t)n * a->chunks * p->groups,
                                          ceil_div(pixels, kTile) * ceil_div(p->channels, kTile) * n);
    if (wgs > 0x7fffffff) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "group norm: tensor too large");
  }
  return ok();
}

template <class T, int ACT>
int norm_apply(const NormArgs& a, int layout, int n, bool vec, hipStream_t s) {
  if (layout == NHIP_LAYOUT_BLOBS) {
    const int pt = (int)ceil_div(a.pixels, kTile), ct = (int)ceil_div(a.channels, kTile);
    NHIP_LAUNCH("group_norm_apply", (norm_apply_blobs_kernel<T, ACT>), dim3((uint32_t)((int64_t)pt * ct * n)),
                dim3(kBlobThreads), 0, s, a, pt, ct);
  } else {
    // Many chunks to merge: a workgroup takes fewer groups (of 256 bytes of a
    // pixel at least) and as many more chunks.  us a call without / with this:
    // 4 x 4096 x 320 bf16 (128 chunks) 22.6 / 19.0, 1 x 12544 x 320 fp32 (256)
    // 27.5 / 19.8; of 64 chunks 8 x 50175 x 320 172 / 180.
    constexpr int V = kVec<T>;
    int each = a.groups;
    if (a.chunks > 64)
      while (each % 2 == 0 && each / 2 * a.cpg * (int)sizeof(T) >= 256 && (!vec || each / 2 * a.cpg % V == 0)) each /= 2;
    const int run = a.groups / each, runs = (int)ceil_div(a.chunks, run);
    const dim3 grid((uint32_t)((int64_t)n * runs * run));
    const auto launch = [&](auto kernel) {
      NHIP_LAUNCH("group_norm_apply", kernel, grid, dim3(kThreads), each * sizeof(float2), s, a, each, run, runs);
    };
    if (vec)
      // us without / with: 257 MB 165 / 144, 128 MB 87 / 73, 103 MB 69 / 57, 51 MB 33.0 / 32.7
      n * a.pixels * a.channels * (int64_t)sizeof(T) > kStreamBytes ? launch(norm_apply_tokens_kernel<T, V, ACT, true>) : launch(norm_apply_tokens_kernel<T, V, ACT, false>);
    else
      launch(norm_apply_tokens_kernel<T, 1, ACT, false>);
  }
  return check_launch("group_norm_apply");
}

// Channels' moments and the threads' sums.
size_t stats_lds(int channels, int v, int threads) {
  return channels * sizeof(double2) + sums_place(v, threads) * sizeof(double);
}

template <class T, int ACT>
int norm_one(const NormArgs& a, int layout, int n, int groups, bool vec, hipStream_t s) {
  constexpr int V = kVec<T>;
  const dim3 grid((uint32_t)((int64_t)n * (a.groups / groups)));
  if (layout == NHIP_LAYOUT_BLOBS) {
    if (vec)
      NHIP_LAUNCH("group_norm_one", (norm_one_blobs_kernel<T, V, ACT>), grid, dim3(kOneThreads), 0, s, a, fast_div(a.cpg));
    else
      NHIP_LAUNCH("group_norm_one", (norm_one_blobs_kernel<T, 1, ACT>), grid, dim3(kOneThreads), 0, s, a, fast_div(a.cpg));
  } else {
    const bool wide = vec && groups * a.cpg % V == 0;
    const size_t lds = stats_lds(groups * a.cpg, wide ? V : 1, kOneThreads);
    const void* kernel = wide ? (const void*)norm_one_tokens_kernel<T, V, ACT> : (const void*)norm_one_tokens_kernel<T, 1, ACT>;
    if (lds > 65536) NHIP_TRY(ensure_dynamic_lds(kernel, 160 * 1024));
    if (wide)
      NHIP_LAUNCH("group_norm_one", (norm_one_tokens_kernel<T, V, ACT>), grid, dim3(kOneThreads), lds, s, a, groups);
    else
      NHIP_LAUNCH("group_norm_one", (norm_one_tokens_kernel<T, 1, ACT>), grid, dim3(kOneThreads), lds, s, a, groups);
  }
  return check_launch("group_norm_one");
}

// Groups that a workgroup which holds their values does, and its threads
// (tokens of whole 16-byte vectors): groups whose channels fill 64 bytes of a
// pixel, more of them where threads and workgroups are left.  0: not here.
//
// us a call, two launches / held.  Of 256 or 512 threads, several to a CU: 64 x
// 784 x 512 bf16 34.7 / 25.2, 128 x 55.6 / 40.3, 32 x fp32 31.2 / 21.8, 16 x
// 1024 x 1280 f16 32.5 / 23.4; of 512 threads and 8 / 64 workgroups 11.2 / 12.0,
// 14.9 / 12.6.  Rows that are no whole 64 bytes share lines with their
// neighbours, which costs where results are past the caches: 1024 x 640 f16 of 42
// MB 30.2 / 23.4, of 84 45.7 / 55.2 or, another time, 48.0 / 43.1.  Of 1024 threads,
// one to a CU, with nothing beside its waits: 3136 x 256 bf16 of 128 / 192 / 256 / 384
// / 512 / 1024 workgroups 22.6 / 23.5, 34.2 / 25.1, 33.2 / 26.8, 53.5 / 47.8, 54.6 /
// 53.4, 111 / 115.
struct Held {
  int groups, threads;
};
Held groups_held(const NormArgs& a, int n, int es) {
  const int force = setting_int("NHIP_NORM_ONE", -1);
  if (force == 0 || force == 1) return {0, 0};
  const auto threads_of = [&](int each) {
    const int cols = each * a.cpg * es / 16;
    for (int th : {256, 512, 1024})
      if (cols <= th && a.pixels <= (int64_t)kHeld * (th / cols)) return th;
    return 0;
  };
  int each = 1;
  while ((each * a.cpg * es < 64 || each * a.cpg * es % 16) && a.groups % (2 * each) == 0) each *= 2;
  if (each * a.cpg * es % 16 || !threads_of(each)) return {0, 0};
  while (a.groups % (2 * each) == 0 && threads_of(2 * each) == 256 && (int64_t)n * (a.groups / (2 * each)) >= 4 * cu_count()) each *= 2;
  const int64_t wgs = (int64_t)n * (a.groups / each);
  if (wgs > 0x7fffff00) return {0, 0};
  const Held held{each, threads_of(each)};
  if (force == 2) return held;
  if (each * a.cpg * es % 64 && n * a.pixels * a.channels * es > kStreamBytes) return {0, 0};
  if (held.threads == 512 && wgs * 4 < cu_count()) return {0, 0};
  if (held.threads == 1024 && (wgs * 4 < 3 * cu_count() || wgs > 2 * cu_count())) return {0, 0};
  return held;
}

template <class T, int ACT, int TH>
int norm_held(const NormArgs& a, int n, int groups, hipStream_t s) {
  constexpr int V = kVec<T>;
  const int wgs = n * (a.groups / groups);
  const size_t lds = stats_lds(groups * a.cpg, V, TH);
  const auto launch = [&](auto kernel) {
    if (lds > 65536) {
      const int st = ensure_dynamic_lds((const void*)kernel, 160 * 1024);
      if (st != NHIP_STATUS_SUCCESS) return st;
    }
    NHIP_LAUNCH("group_norm_held", kernel, dim3((uint32_t)ceil_div(wgs, 8) * 8), dim3(TH), lds, s, a, groups, wgs);
    return check_launch("group_norm_held");
  };
  const bool stream = n * a.pixels * a.channels * (int64_t)sizeof(T) > kStreamBytes && groups * a.cpg * sizeof(T) % 64 == 0;
  return stream ? launch(norm_held_tokens_kernel<T, V, ACT, TH, true>) : launch(norm_held_tokens_kernel<T, V, ACT, TH, false>);
}

template <class T, int ACT>
int norm_held(const NormArgs& a, int n, Held held, hipStream_t s) {
  switch (held.threads) {
    case 256: return norm_held<T, ACT, 256>(a, n, held.groups, s);
    case 512: return norm_held<T, ACT, 512>(a, n, held.groups, s);
    default: return norm_held<T, ACT, 1024>(a, n, held.groups, s);
  }
}

template <class T>
int norm_run(const NormArgs& a, int layout, int n, int one, hipStream_t s) {
  constexpr int V = kVec<T>;
  const bool blobs = layout == NHIP_LAYOUT_BLOBS;
  // whole 16-byte vectors: along the pixels (blobs) or the channels (tokens)
  const bool vec = aligned_to(a.x, 16) && a.image_stride % V == 0 && a.row_stride % V == 0 &&
                   (blobs ? a.pixels % V == 0 : a.channels % V == 0 && aligned_to(a.y, 16));
  if (one) switch (a.act) {
      case NHIP_ACT_RELU: return norm_one<T, NHIP_ACT_RELU>(a, layout, n, one, vec, s);
      case NHIP_ACT_SILU: return norm_one<T, NHIP_ACT_SILU>(a, layout, n, one, vec, s);
      default: return norm_one<T, NHIP_ACT_NONE>(a, layout, n, one, vec, s);
    }
  if (const Held held = !blobs && vec ? groups_held(a, n, sizeof(T)) : Held{0, 0}; held.groups) switch (a.act) {
      case NHIP_ACT_RELU: return norm_held<T, NHIP_ACT_RELU>(a, n, held, s);
      case NHIP_ACT_SILU: return norm_held<T, NHIP_ACT_SILU>(a, n, held, s);
      default: return norm_held<T, NHIP_ACT_NONE>(a, n, held, s);
    }
  if (blobs) {
    const dim3 grid((uint32_t)((int64_t)n * a.chunks * a.groups));
    if (vec)
      NHIP_LAUNCH("group_norm_stats", (norm_stats_blobs_kernel<T, V>), grid, dim3(kBlobThreads), 0, s, a);
    else
      NHIP_LAUNCH("group_norm_stats", (norm_stats_blobs_kernel<T, 1>), grid, dim3(kBlobThreads), 0, s, a);
  } else {
    const dim3 grid((uint32_t)(n * a.chunks));
    const size_t lds = stats_lds(a.channels, vec ? V : 1, kThreads);
    const auto launch = [&](auto kernel) {
      if (lds > 65536) {
        const int st = ensure_dynamic_lds((const void*)kernel, 160 * 1024);
        if (st != NHIP_STATUS_SUCCESS) return st;
      }
      NHIP_LAUNCH("group_norm_stats", kernel, grid, dim3(kThreads), lds, s, a);
      return ok();
    };
    NHIP_TRY(vec ? launch(norm_stats_tokens_kernel<T, V>) : launch(norm_stats_tokens_kernel<T, 1>));
  }
  NHIP_TRY(check_launch("group_norm_stats"));
  switch (a.act) {
    case NHIP_ACT_RELU: return norm_apply<T, NHIP_ACT_RELU>(a, layout, n, vec, s);
    case NHIP_ACT_SILU: return norm_apply<T, NHIP_ACT_SILU>(a, layout, n, vec, s);
    default: return norm_apply<T, NHIP_ACT_NONE>(a, layout, n, vec, s);
  }
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int nhip_group_norm_create(int32_t channels, int32_t groups, const float* gamma, const float* beta, float eps,
                           int32_t activation, nhip_norm_t* plan) {
  if (!plan) return fail(NHIP_STATUS_NULL_POINTER, "group norm: null plan pointer");
  *plan = nullptr;
  if (!gamma != !beta) return fail(NHIP_STATUS_NULL_POINTER, "group norm: gamma and beta come together");
  if (channels <= 0 || groups <= 0 || channels % groups || channels > kMaxChannels)
    return fail(NHIP_STATUS_INVALID_SHAPE, "group norm: channels have to be a multiple of groups, 4096 at most");
  if (!(eps >= 0.f) || eps > 3e38f) return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "group norm: eps has to be finite, 0 or more");
  if (activation != NHIP_ACT_NONE && activation != NHIP_ACT_RELU && activation != NHIP_ACT_SILU)
    return fail(NHIP_STATUS_UNSUPPORTED, "group norm: activation has to be NONE, RELU or SILU");
  float* dev = nullptr;
  const size_t bytes = 2 * (size_t)channels * sizeof(float);
  try {
    std::vector<float> host(2 * (size_t)channels, 0.f);
    std::fill(host.begin(), host.begin() + channels, 1.f);
    if (gamma) {
      std::copy(gamma, gamma + channels, host.begin());
      std::copy(beta, beta + channels, host.begin() + channels);
    }
    NHIP_TRY(check_hip(hipMalloc(reinterpret_cast<void**>(&dev), bytes), "hipMalloc(group norm)"));
    const int st = check_hip(hipMemcpy(dev, host.data(), bytes, hipMemcpyHostToDevice), "hipMemcpy(group norm)");
    if (st != NHIP_STATUS_SUCCESS) {
      (void)hipFree(dev);
      return st;
    }
    nhip_norm_plan* p = new nhip_norm_plan;
    p->channels = channels;
    p->groups = groups;
    p->act = activation;
    p->eps = eps;
    p->affine = dev;
    *plan = p;
  } catch (const std::bad_alloc&) {
    (void)hipFree(dev);
    return fail(NHIP_STATUS_DEVICE_ERROR, "group norm: out of host memory");
  }
  return ok();
}

int nhip_group_norm_workspace_size(nhip_norm_t plan, int32_t dtype, int32_t layout, int32_t n, int64_t pixels,
                                   uint64_t* bytes) {
  if (!bytes) return fail(NHIP_STATUS_NULL_POINTER, "group norm: null pointer");
  NormArgs a{};
  int one;
  NHIP_TRY(norm_args(plan, dtype, layout, n, pixels, &a, &one));
  *bytes = (uint64_t)n * a.chunks * a.groups * sizeof(double2);
  return ok();
}

int nhip_group_norm_forward(nhip_norm_t plan, const void* input, int32_t dtype, int32_t layout, int32_t n,
                            int64_t pixels, int64_t image_stride, int64_t row_stride, void* output, void* workspace,
                            uint64_t workspace_bytes, void* stream) {
  NormArgs a{};
  int one;
  NHIP_TRY(norm_args(plan, dtype, layout, n, pixels, &a, &one));
  if (n == 0 || pixels == 0) return ok();
  if (!input || !output) return fail(NHIP_STATUS_NULL_POINTER, "group norm: null pointer");
  const int es = elem_size(dtype);
  if (!aligned_to(input, es) || !aligned_to(output, es))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "group norm: a tensor is not aligned to its type");
  if (row_stride < (layout == NHIP_LAYOUT_BLOBS ? pixels : (int64_t)a.channels) || image_stride < 0)
    return fail(NHIP_STATUS_INVALID_SHAPE, "group norm: rows overlap");
  const uint64_t need = (uint64_t)n * a.chunks * a.groups * sizeof(double2);
  if (need && !workspace) return fail(NHIP_STATUS_NULL_POINTER, "group norm: null workspace");
  if (need && (workspace_bytes < need || !aligned_to(workspace, 16)))
    return fail(NHIP_STATUS_OUTPUT_CAPACITY_INSUFFICIENT, "group norm: workspace too small or not 16-byte aligned");
  a.x = input;
  a.y = output;
  a.part = (double2*)workspace;
  a.image_stride = image_stride;
  a.row_stride = row_stride;
  return NHIP_FOR_ELEM(dtype, T, norm_run<T>(a, layout, n, one, as_stream(stream)));
}

int nhip_norm_destroy(nhip_norm_t plan) {
  if (!plan) return ok();
  (void)hipFree(plan->affine);
  delete plan;
  return ok();
}

}  // extern "C"
