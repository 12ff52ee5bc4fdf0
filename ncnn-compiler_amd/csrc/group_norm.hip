// Group norm with an activation into channels-last tokens:
//   y = act((x - mean_g) / sqrt(var_g + eps) * gamma_c + beta_c).
//
// Two launches: the statistics of every (image, group) over chunks of pixels
// (a mean and a sum of squared deviations each), and a pass that merges them
// and writes y.  Both stream the tensor, so bytes bound them: x is read
// twice, the second time from the last-level cache where the tensor fits.
//
// Statistics: sums of x - s and (x - s)^2 with s one of the values summed, over
// at most a few hundred terms of a thread; means and squared deviations of
// channels and chunks are then merged in 64 bits (the sum of squares about a
// common mean is the sum of the parts' plus count * (difference of means)^2).
// A large mean beside a small spread therefore loses nothing, as it would in
// E[x^2] - E[x]^2.  A thread's sums are fp32; those of fp32 values' first
// powers are 64 bits, so that results near 0 keep their digits (an element
// costs a conversion and an addition more, hidden behind its four bytes).
#include <algorithm>
#include <new>
#include <vector>

#include "elem.h"

struct nhip_norm_plan {
  int32_t channels, groups, act;
  float eps;
  float* affine = nullptr;  // gamma [channels], beta [channels]
};

namespace nhip {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxChannels = 4096;
constexpr int kMaxChunks = 128;  // parts of an image: what each workgroup of the second pass merges
constexpr int kTile = 64;        // pixels and channels of a transposed tile (blobs)

struct NormArgs {
  const void* x;
  void* y;
  double2* part;  // [n][chunks][groups]: mean, sum of squared deviations
  const float* affine;
  int64_t pixels, image_stride, row_stride;
  int channels, groups, cpg, act;
  int chunks;           // of an image
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
__device__ __forceinline__ int team_of(int groups) {
  int t = 64;
  while (t > 1 && (kThreads / t) < groups) t >>= 1;
  return t;
}
template <class S>
__device__ __forceinline__ S team_sum(S v, int team) {
  for (int o = team >> 1; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// What a thread sums first powers in.
template <class T>
struct First {
  typedef float type;
};
template <>
struct First<float> {
  typedef double type;
};
// The value whose first powers are summed: x itself in 64 bits, else x - s.
__device__ __forceinline__ float first_power(float x, float d, float) { return d; }
__device__ __forceinline__ double first_power(float x, float d, double) { return (double)x; }
// Mean and squared deviations of `count` values from their sums.
__device__ __forceinline__ double2 moments(float s1, float s2, float shift, double count) {
  const double d = (double)s1 / count;
  return make_double2((double)shift + d, fmax((double)s2 - (double)s1 * d, 0.0));
}
__device__ __forceinline__ double2 moments(double s1, float s2, float shift, double count) {
  const double mean = s1 / count, d = mean - (double)shift;
  return make_double2(mean, fmax((double)s2 - count * d * d, 0.0));
}

// Merges the chunks of image `n` for groups [g0, g1): mean and 1/sqrt(var + eps)
// to stat[g - g0].
__device__ void merge_chunks(const NormArgs& a, int n, int g0, int g1, float2* stat) {
  const int team = team_of(g1 - g0), lane = threadIdx.x & (team - 1);
  const double2* part = a.part + (int64_t)n * a.chunks * a.groups;
  const double last = (double)(a.pixels - (int64_t)(a.chunks - 1) * a.chunk), total = (double)a.pixels;
  for (int gb = g0; gb < g1; gb += kThreads / team) {  // uniform: all lanes of a team stay in the butterflies
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

// Statistics of one chunk of one image, channels last.  A thread keeps its V
// channels and walks pixels; channels are merged into groups through LDS.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void norm_stats_tokens_kernel(NormArgs a) {
  typedef typename First<T>::type S;
  extern __shared__ double2 lds[];  // [channels] mean, deviations; then [threads][V] first, [threads][V] second sums
  S* red1 = reinterpret_cast<S*>(lds + a.channels);
  float* red2 = reinterpret_cast<float*>(red1 + kThreads * V);
  const int n = blockIdx.x / a.chunks, k = blockIdx.x % a.chunks;
  const int64_t p0 = (int64_t)k * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
  const T* x = (const T*)a.x + n * a.image_stride;
  const int vecs = a.channels / V;
  const double count = (double)(p1 - p0);
  for (int v0 = 0; v0 < vecs; v0 += kThreads) {
    const int cols = min(kThreads, vecs - v0), rows = kThreads / cols;
    const int col = threadIdx.x % cols, row = threadIdx.x / cols;
    S s1[V] = {};
    float s2[V] = {}, shift[V];
    if (row < rows) {
      const T* px = x + (int64_t)(v0 + col) * V;
      Vec<T, V>::load(px + p0 * a.row_stride, shift);
#pragma unroll 4
      for (int64_t p = p0 + row; p < p1; p += rows) {
        float t[V];
        Vec<T, V>::load(px + p * a.row_stride, t);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = t[i] - shift[i];
          s1[i] += first_power(t[i], d, S());
          s2[i] = fmaf(d, d, s2[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        red1[(row * cols + col) * V + i] = s1[i];
        red2[(row * cols + col) * V + i] = s2[i];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols * V; c += kThreads) {
      S u1 = 0;
      float u2 = 0.f;
      for (int r = 0; r < rows; ++r) {
        u1 += red1[r * cols * V + c];
        u2 += red2[r * cols * V + c];
      }
      lds[v0 * V + c] = moments(u1, u2, (float)x[p0 * a.row_stride + v0 * V + c], count);
    }
    __syncthreads();
  }
  const int team = team_of(a.groups), lane = threadIdx.x & (team - 1);
  for (int gb = 0; gb < a.groups; gb += kThreads / team) {
    const int g = gb + threadIdx.x / team;
    const bool in = g < a.groups;
    const double2* ch = lds + g * a.cpg;
    double m = 0.0;
    for (int c = lane; in && c < a.cpg; c += team) m += ch[c].x;
    m = team_sum(m, team) / a.cpg;
    double v = 0.0;
    for (int c = lane; in && c < a.cpg; c += team) {
      const double d = ch[c].x - m;
      v += ch[c].y + count * d * d;
    }
    v = team_sum(v, team);
    if (in && lane == 0) a.part[(int64_t)blockIdx.x * a.groups + g] = make_double2(m, v);
  }
}

template <class T, int V, int ACT>
__global__ __launch_bounds__(kThreads) void norm_apply_tokens_kernel(NormArgs a) {
  extern __shared__ float2 stats[];  // [groups]
  const int n = blockIdx.x / a.chunks, k = blockIdx.x % a.chunks;
  merge_chunks(a, n, 0, a.groups, stats);
  __syncthreads();
  const int64_t p0 = (int64_t)k * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
  const T* x = (const T*)a.x + n * a.image_stride;
  T* y = (T*)a.y + n * a.pixels * a.channels;
  const int vecs = a.channels / V;
  for (int v0 = 0; v0 < vecs; v0 += kThreads) {
    const int cols = min(kThreads, vecs - v0), rows = kThreads / cols;
    const int col = threadIdx.x % cols, row = threadIdx.x / cols;
    if (row >= rows) continue;
    const int c0 = (v0 + col) * V;
    float mean[V], scale[V], beta[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float2 s = stats[(c0 + i) / a.cpg];
      mean[i] = s.x;
      scale[i] = s.y * a.affine[c0 + i];
      beta[i] = a.affine[a.channels + c0 + i];
    }
#pragma unroll 4
    for (int64_t p = p0 + row; p < p1; p += rows) {
      float t[V];
      Vec<T, V>::load(x + p * a.row_stride + c0, t);
#pragma unroll
      for (int i = 0; i < V; ++i) t[i] = activate<ACT>(fmaf(t[i] - mean[i], scale[i], beta[i]));
      Vec<T, V>::store(y + p * a.channels + c0, t);
    }
  }
}

// Statistics of one chunk of pixels of one group, channels first.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void norm_stats_blobs_kernel(NormArgs a) {
  typedef typename First<T>::type S;
  __shared__ S red1[kThreads / 64];
  __shared__ float red2[kThreads / 64];
  const int g = blockIdx.x % a.groups, nk = blockIdx.x / a.groups;
  const int n = nk / a.chunks, k = nk % a.chunks;
  const int64_t p0 = (int64_t)k * a.chunk, p1 = min(p0 + a.chunk, a.pixels);
  const T* x = (const T*)a.x + n * a.image_stride + (int64_t)g * a.cpg * a.row_stride;
  const float shift = (float)x[p0];
  const int vecs = (int)((p1 - p0) / V);
  S s1 = 0;
  float s2 = 0.f;
  const int lanes = min(kThreads, (vecs + 63) / 64 * 64);
  const int rows = kThreads / lanes, row = threadIdx.x / lanes, col = threadIdx.x % lanes;
  if (row < rows)
    for (int c = row; c < a.cpg; c += rows)
      for (int v = col; v < vecs; v += lanes) {
        float t[V];
        Vec<T, V>::load(x + c * a.row_stride + p0 + (int64_t)v * V, t);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float d = t[i] - shift;
          s1 += first_power(t[i], d, S());
          s2 = fmaf(d, d, s2);
        }
      }
  s1 = team_sum(s1, 64);
  s2 = team_sum(s2, 64);
  if ((threadIdx.x & 63) == 0) {
    red1[threadIdx.x / 64] = s1;
    red2[threadIdx.x / 64] = s2;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    S u1 = 0;
    float u2 = 0.f;
    for (int i = 0; i < kThreads / 64; ++i) {
      u1 += red1[i];
      u2 += red2[i];
    }
    a.part[(int64_t)nk * a.groups + g] = moments(u1, u2, shift, (double)(p1 - p0) * a.cpg);
  }
}

// A tile of kTile channels x kTile pixels through LDS: read along the pixels,
// written along the channels.
template <class T, int ACT>
__global__ __launch_bounds__(kThreads) void norm_apply_blobs_kernel(NormArgs a, int ptiles, int ctiles) {
  __shared__ float tile[kTile][kTile + 1];
  __shared__ float2 stat[kTile];
  const int pt = blockIdx.x % ptiles, rest = blockIdx.x / ptiles;
  const int c0 = rest % ctiles * kTile, n = rest / ctiles;
  const int64_t p0 = (int64_t)pt * kTile;
  const int cn = min(kTile, a.channels - c0), pn = (int)min((int64_t)kTile, a.pixels - p0);
  const int g0 = c0 / a.cpg, g1 = (c0 + cn - 1) / a.cpg + 1;
  merge_chunks(a, n, g0, g1, stat);
  const T* x = (const T*)a.x + n * a.image_stride + p0;
  T* y = (T*)a.y + (n * a.pixels + p0) * a.channels + c0;
  const int lane = threadIdx.x % kTile, row = threadIdx.x / kTile;
#pragma unroll 4
  for (int c = row; c < cn; c += kThreads / kTile)
    if (lane < pn) tile[c][lane] = (float)x[(int64_t)(c0 + c) * a.row_stride + lane];
  __syncthreads();
  if (lane >= cn) return;
  const float2 s = stat[(c0 + lane) / a.cpg - g0];
  const float scale = s.y * a.affine[c0 + lane], beta = a.affine[a.channels + c0 + lane];
#pragma unroll 4
  for (int p = row; p < pn; p += kThreads / kTile)
    y[(int64_t)p * a.channels + lane] = (T)activate<ACT>(fmaf(tile[lane][p] - s.x, scale, beta));
}

// Chunks of an image: enough workgroups for four to a CU, each of at least
// 8192 values, and few enough to be merged by every workgroup of the second
// pass.
void chunks_of(int channels, int64_t n, int64_t pixels, int per_image, NormArgs* a) {
  const int64_t want = ceil_div((int64_t)4 * cu_count(), n * per_image);
  const int64_t fit = std::max<int64_t>(1, pixels * channels / per_image / 8192);
  int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({want, fit, (int64_t)kMaxChunks, pixels}));
  a->chunk = round_up(ceil_div(pixels, chunks), 8);  // whole vectors along the pixels (blobs)
  a->chunks = (int)ceil_div(pixels, a->chunk);
}

int norm_args(const nhip_norm_plan* p, int32_t dtype, int32_t layout, int32_t n, int64_t pixels, NormArgs* a) {
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
  if (n && pixels) {
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
                dim3(kThreads), 0, s, a, pt, ct);
  } else if (vec) {
    NHIP_LAUNCH("group_norm_apply", (norm_apply_tokens_kernel<T, kVec<T>, ACT>), dim3((uint32_t)(n * a.chunks)),
                dim3(kThreads), a.groups * sizeof(float2), s, a);
  } else {
    NHIP_LAUNCH("group_norm_apply", (norm_apply_tokens_kernel<T, 1, ACT>), dim3((uint32_t)(n * a.chunks)),
                dim3(kThreads), a.groups * sizeof(float2), s, a);
  }
  return check_launch("group_norm_apply");
}

template <class T>
size_t stats_lds(int channels, int v) {
  return channels * sizeof(double2) + kThreads * v * (sizeof(typename First<T>::type) + sizeof(float));
}

template <class T>
int norm_run(const NormArgs& a, int layout, int n, hipStream_t s) {
  constexpr int V = kVec<T>;
  const bool blobs = layout == NHIP_LAYOUT_BLOBS;
  // whole 16-byte vectors: along the pixels (blobs) or the channels (tokens)
  const bool vec = aligned_to(a.x, 16) && a.image_stride % V == 0 && a.row_stride % V == 0 &&
                   (blobs ? a.pixels % V == 0 : a.channels % V == 0 && aligned_to(a.y, 16));
  if (blobs) {
    const dim3 grid((uint32_t)((int64_t)n * a.chunks * a.groups));
    if (vec)
      NHIP_LAUNCH("group_norm_stats", (norm_stats_blobs_kernel<T, V>), grid, dim3(kThreads), 0, s, a);
    else
      NHIP_LAUNCH("group_norm_stats", (norm_stats_blobs_kernel<T, 1>), grid, dim3(kThreads), 0, s, a);
  } else {
    const dim3 grid((uint32_t)(n * a.chunks));
    if (vec)
      NHIP_LAUNCH("group_norm_stats", (norm_stats_tokens_kernel<T, V>), grid, dim3(kThreads),
                  stats_lds<T>(a.channels, V), s, a);
    else
      NHIP_LAUNCH("group_norm_stats", (norm_stats_tokens_kernel<T, 1>), grid, dim3(kThreads),
                  stats_lds<T>(a.channels, 1), s, a);
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
  NHIP_TRY(norm_args(plan, dtype, layout, n, pixels, &a));
  *bytes = (uint64_t)n * a.chunks * a.groups * sizeof(double2);
  return ok();
}

int nhip_group_norm_forward(nhip_norm_t plan, const void* input, int32_t dtype, int32_t layout, int32_t n,
                            int64_t pixels, int64_t image_stride, int64_t row_stride, void* output, void* workspace,
                            uint64_t workspace_bytes, void* stream) {
  NormArgs a{};
  NHIP_TRY(norm_args(plan, dtype, layout, n, pixels, &a));
  if (n == 0 || pixels == 0) return ok();
  if (!input || !output) return fail(NHIP_STATUS_NULL_POINTER, "group norm: null pointer");
  const int es = elem_size(dtype);
  if (!aligned_to(input, es) || !aligned_to(output, es))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "group norm: a tensor is not aligned to its type");
  if (row_stride < (layout == NHIP_LAYOUT_BLOBS ? pixels : (int64_t)a.channels) || image_stride < 0)
    return fail(NHIP_STATUS_INVALID_SHAPE, "group norm: rows overlap");
  const uint64_t need = (uint64_t)n * a.chunks * a.groups * sizeof(double2);
  if (!workspace) return fail(NHIP_STATUS_NULL_POINTER, "group norm: null workspace");
  if (workspace_bytes < need || !aligned_to(workspace, 16))
    return fail(NHIP_STATUS_OUTPUT_CAPACITY_INSUFFICIENT, "group norm: workspace too small or not 16-byte aligned");
  a.x = input;
  a.y = output;
  a.part = (double2*)workspace;
  a.image_stride = image_stride;
  a.row_stride = row_stride;
  return NHIP_FOR_ELEM(dtype, T, norm_run<T>(a, layout, n, as_stream(stream)));
}

int nhip_norm_destroy(nhip_norm_t plan) {
  if (!plan) return ok();
  (void)hipFree(plan->affine);
  delete plan;
  return ok();
}

}  // extern "C"
