// The 8-bit cache of keys and values: tokens quantised into pages with a
// scale for each page and head, and read back as values.  (The attention over
// it: attention.h.)
//
// Compiled with -ffp-contract=off: a code is the rounding of one separately
// rounded product, so that it can be restated bit for bit.
#include <algorithm>
#include <type_traits>

#include "elem.h"
#include "kv_cache8.h"

namespace nhip {
namespace {

constexpr int kThreads = 256;  // of a workgroup that reads
constexpr int kHeld = 4;       // vectors that a thread appends without reading them again

struct AppendArgs {
  Kv8 c;
  const void* x[2];      // keys, values
  int64_t xs[2][3];      // batch, token, head
  const int32_t* starts;
  const int32_t* counts;
  int32_t tokens, touch;  // pages that a sequence may touch
  FastDiv by_vecs;        // vectors of a token's head
};

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// One workgroup: one page of one sequence, one head, keys or values.  The new
// tokens are wanted twice, for their largest magnitude and to be quantised: a
// thread keeps its first kHeld vectors and reads others again.  Bytes bound
// it: 4 x 3136 tokens of 8 heads of 128 bf16 17.5 us (77 MB, 4.4 TB/s; a
// workgroup's loads, its maximum and its stores wait for each other); one token
// to each of 64 sequences 4.4 us, where a workgroup is one wave.  (Pages whose
// scale stands.  Where it grows at every call, and the 41 tokens that a page holds
// are requantised: 8.3 us a call instead of 6.7 for the single tokens.)
template <class T, int V, int TH>
__global__ __launch_bounds__(TH) void kv8_append_kernel(AppendArgs a) {
  const int which = blockIdx.x & 1;
  const uint32_t rest = blockIdx.x >> 1;
  const int h = rest % a.c.kv_heads;
  const uint32_t rest2 = rest / a.c.kv_heads;
  const int j = rest2 % a.touch, b = rest2 / a.touch;
  const int start = a.starts[b];
  const int count = a.counts ? min(a.counts[b], a.tokens) : a.tokens;
  if (start < 0 || count <= 0) return;
  const int64_t page = (int64_t)(start >> a.c.shift) + j;
  const int64_t t0 = max((int64_t)start, page << a.c.shift);
  const int64_t t1 = min((int64_t)start + count, (page + 1) << a.c.shift);
  if (t0 >= t1) return;
  const int d = a.c.head_dim;
  const T* x = (const T*)a.x[which] + b * a.xs[which][0] + (t0 - start) * a.xs[which][1] + h * a.xs[which][2];
  const int64_t xt = a.xs[which][1];
  const int vecs = d / V, fresh = (int)(t1 - t0) * vecs;
  const auto load = [&](int i, float(&t)[V]) {
    const int token = fdiv(i, a.by_vecs);
    Vec<T, V>::load(x + token * xt + (i - token * vecs) * V, t);
  };
  float held[kHeld][V];
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (const int i = threadIdx.x + k * TH; i < fresh) load(i, held[k]);
  const int64_t id = kv8_page(a.c, b, page);
  if (id < 0) return;
  int8_t* code = (which ? a.c.v : a.c.k) + ((id * a.c.kv_heads + h) << a.c.shift) * d;
  float* scale = (which ? a.c.v_scale : a.c.k_scale) + id * a.c.kv_heads + h;
  const int had = (int)(t0 - (page << a.c.shift));  // tokens that the page holds
  const float stood = *scale;

  // the largest magnitude; NaN does not count, infinities only if asked for
  const auto largest = [&](auto any) {
    float most = 0.f;
    const auto widest = [&](const float(&t)[V]) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float m = fabsf(t[e]);
        most = any() || m <= 3.402823466e38f ? fmaxf(most, m) : most;
      }
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (threadIdx.x + k * TH < fresh) widest(held[k]);
    for (int i = threadIdx.x + kHeld * TH; i < fresh; i += TH) {
      float t[V];
      load(i, t);
      widest(t);
    }
    most = wave_max(most);
    if constexpr (TH > 64) {
      __shared__ float red[TH / 64];
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x / 64] = most;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < TH / 64; ++i) most = fmaxf(most, red[i]);
    }
    return most;
  };
  // (two instructions less a value than without infinities at once: 19.9 -> 17.5 us)
  float most = largest(std::true_type());
  if (__builtin_expect(most > 3.402823466e38f, false)) most = largest(std::false_type());
  const float was = had ? stood : 0.f;
  const float want = most > 0.f ? fmaxf(most * (1.0f / 127.0f), kScaleLeast) : 0.f;
  const float now = fmaxf(want, was);
  const float inv = now > 0.f ? 1.0f / now : 0.f;
  if (threadIdx.x == 0) *scale = now;  // (every lane's own read of it is done: `now` depends on it)
  if (now != was) {
    const float ratio = was * inv;
    uint2* old = reinterpret_cast<uint2*>(code);  // head_dim is a multiple of 8
    for (int i = threadIdx.x; i < had * d / 8; i += TH) {
      const uint2 c = old[i];
      int q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = quantize_q((float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3))), ratio);
      old[i] = make_uint2(pack_i8x4(q[0], q[1], q[2], q[3]), pack_i8x4(q[4], q[5], q[6], q[7]));
    }
  }
  int8_t* to = code + had * d;
  const auto put = [&](int i, const float(&t)[V]) {
    int q[V];
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = quantize_q(t[e], inv);
    if constexpr (V >= 4) {
#pragma unroll
      for (int e = 0; e < V; e += 4)
        reinterpret_cast<uint32_t*>(to + i * V)[e / 4] = pack_i8x4(q[e], q[e + 1], q[e + 2], q[e + 3]);
    } else {
      to[i] = (int8_t)q[0];
    }
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (const int i = threadIdx.x + k * TH; i < fresh) put(i, held[k]);
  for (int i = threadIdx.x + kHeld * TH; i < fresh; i += TH) {
    float t[V];
    load(i, t);
    put(i, t);
  }
}

struct ReadArgs {
  Kv8 c;
  void* out[2];
  const int32_t* starts;
  int32_t tokens, items, blocks;  // of a sequence: 8-channel pieces, workgroups
  FastDiv by_vecs, by_heads;
};

// A thread: eight channels of one token and head, keys and values, for which
// the page is found once (us with a thread for each / for both: bf16 15.7 / 14.9,
// fp32 23.7 / 24.4, small reads 9.1 / 8.6).  Bytes bound it: 4 x 3136 tokens of 8
// heads of 128 to bf16 15 us (77 MB, 5.1 TB/s, as a large copy).
template <class T>
__global__ __launch_bounds__(kThreads) void kv8_read_kernel(ReadArgs a) {
  const uint32_t block = blockIdx.x;
  const int b = block / a.blocks;
  const int i = (int)(block % a.blocks) * kThreads + threadIdx.x;
  if (i >= a.items) return;
  const int r = fdiv(i, a.by_vecs), c = (i - r * (a.c.head_dim / 8)) * 8;
  const int at_token = fdiv(r, a.by_heads), h = r - at_token * a.c.kv_heads;
  const int64_t t = (int64_t)a.starts[b] + at_token;
  const int64_t id = t < 0 ? -1 : kv8_page(a.c, b, t >> a.c.shift);
  float v[2][8] = {};
  if (id >= 0) {
    const int64_t page = id * a.c.kv_heads + h;
    const int64_t at = ((page << a.c.shift) + (t & ((1 << a.c.shift) - 1))) * a.c.head_dim + c;
    const int2 q[2] = {*reinterpret_cast<const int2*>(a.c.k + at), *reinterpret_cast<const int2*>(a.c.v + at)};
    const float s[2] = {a.c.k_scale[page], a.c.v_scale[page]};
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[w][e] = (float)(int8_t)((e < 4 ? q[w].x : q[w].y) >> (8 * (e & 3))) * s[w];
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    T* out = (T*)a.out[w] + ((int64_t)b * a.items + i) * 8;
#pragma unroll
    for (int e = 0; e < 8; e += kVec<T>) Vec<T, kVec<T>>::store(out + e, reinterpret_cast<float(&)[kVec<T>]>(v[w][e]));
  }
}

template <class T, int V>
int append_launch(AppendArgs a, uint32_t wgs, hipStream_t s) {
  const int vecs = a.c.head_dim / V;
  a.by_vecs = fast_div(vecs);
  // As many threads as hold a page's new tokens, 1024 at most; a wave where a
  // call's tokens leave it no more than it holds.  us at 256 / 512 / 1024
  // threads: 4 x 3136 tokens of 8 heads of 128 bf16, pages of 64 (1024 vectors) 17.5 /
  // 19.1 / 28.2; fp32 (2048) 28.2 / 23.3 / 28.2; 2 x 6000 of 4 heads of 256 bf16, pages of
  // 256 (8192) 30.5 / 20.6 / 17.5.
  const int64_t fresh = std::min<int64_t>(a.tokens, int64_t(1) << a.c.shift) * vecs;
  const auto launch = [&](auto kernel, int threads) {
    NHIP_LAUNCH("kv8_append", kernel, dim3(wgs), dim3(threads), 0, s, a);
    return check_launch("kv8_append");
  };
  if ((int64_t)a.tokens * vecs <= kHeld * 64) return launch(kv8_append_kernel<T, V, 64>, 64);
  if (fresh <= kHeld * 256) return launch(kv8_append_kernel<T, V, 256>, 256);
  if (fresh <= kHeld * 512) return launch(kv8_append_kernel<T, V, 512>, 512);
  return launch(kv8_append_kernel<T, V, 1024>, 1024);
}

template <class T>
int append_run(const AppendArgs& a, uint32_t wgs, bool vec, hipStream_t s) {
  return vec ? append_launch<T, kVec<T>>(a, wgs, s) : append_launch<T, 1>(a, wgs, s);
}

template <class T>
int read_run(const ReadArgs& a, uint32_t wgs, hipStream_t s) {
  NHIP_LAUNCH("kv8_read", kv8_read_kernel<T>, dim3(wgs), dim3(kThreads), 0, s, a);
  return check_launch("kv8_read");
}

}  // namespace

int kv8_args(const nhip_kv8_cache* cache, const int32_t* table, int64_t table_pages, Kv8* c) {
  if (!cache) return fail(NHIP_STATUS_NULL_POINTER, "kv8: null cache");
  if (cache->kv_heads <= 0 || cache->pages < 0 || table_pages < 0)
    return fail(NHIP_STATUS_INVALID_SHAPE, "kv8: extents have to be positive");
  if (cache->head_dim <= 0 || cache->head_dim > 256 || cache->head_dim % 8)
    return fail(NHIP_STATUS_INVALID_SHAPE, "kv8: head_dim has to be a multiple of 8, 256 at most");
  int shift = 4;
  while (shift < 8 && (1 << shift) != cache->block_tokens) ++shift;
  if ((1 << shift) != cache->block_tokens)
    return fail(NHIP_STATUS_INVALID_SHAPE, "kv8: block_tokens has to be 16, 32, 64, 128 or 256");
  if (!cache->k || !cache->v || !cache->k_scale || !cache->v_scale || (!table && table_pages))
    return fail(NHIP_STATUS_NULL_POINTER, "kv8: null pointer");
  if (!aligned_to(cache->k, 16) || !aligned_to(cache->v, 16) || !aligned_to(cache->k_scale, 4) ||
      !aligned_to(cache->v_scale, 4) || !aligned_to(table, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "kv8: a tensor is not aligned");
  *c = Kv8{cache->k, cache->v, cache->k_scale, cache->v_scale, table, cache->pages, table_pages,
           cache->kv_heads, cache->head_dim, shift};
  return ok();
}

}  // namespace nhip

using namespace nhip;

extern "C" {

int nhip_kv8_append(const nhip_kv8_cache* cache, int32_t dtype, const void* key, const int64_t* key_strides,
                    const void* value, const int64_t* value_strides, int32_t batch, int32_t tokens,
                    const int32_t* block_table, int64_t table_pages, const int32_t* starts, const int32_t* counts,
                    void* stream) {
  AppendArgs a{};
  NHIP_TRY(kv8_args(cache, block_table, table_pages, &a.c));
  const int es = elem_size(dtype);
  if (!es) return fail(NHIP_STATUS_UNSUPPORTED, "kv8: dtype has to be F32, F16 or BF16");
  if (batch < 0 || tokens < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "kv8: negative extent");
  if (batch == 0 || tokens == 0) return ok();
  if (!key || !value || !key_strides || !value_strides || !starts)
    return fail(NHIP_STATUS_NULL_POINTER, "kv8: null pointer");
  if (!aligned_to(key, es) || !aligned_to(value, es))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "kv8: a tensor is not aligned to its type");
  a.x[0] = key;
  a.x[1] = value;
  const int v = 16 / es;
  bool vec = aligned_to(key, 16) && aligned_to(value, 16);  // head_dim is a multiple of 8
  for (int i = 0; i < 3; ++i) {
    a.xs[0][i] = key_strides[i];
    a.xs[1][i] = value_strides[i];
    if (a.xs[0][i] < 0 || a.xs[1][i] < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "kv8: negative stride");
    vec = vec && a.xs[0][i] % v == 0 && a.xs[1][i] % v == 0;
  }
  a.starts = starts;
  a.counts = counts;
  a.tokens = tokens;
  const int bt = 1 << a.c.shift;
  a.touch = (int)(((int64_t)tokens + bt - 2) / bt + 1);
  const int64_t wgs = (int64_t)batch * a.touch;
  if (wgs > 0x7fffffff / 2 / a.c.kv_heads) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "kv8: too many pages in one call");
  return NHIP_FOR_ELEM(dtype, T, append_run<T>(a, (uint32_t)(wgs * a.c.kv_heads * 2), vec, as_stream(stream)));
}

int nhip_kv8_read(const nhip_kv8_cache* cache, int32_t dtype, int32_t batch, int32_t tokens,
                  const int32_t* block_table, int64_t table_pages, const int32_t* starts, void* key, void* value,
                  void* stream) {
  ReadArgs a{};
  NHIP_TRY(kv8_args(cache, block_table, table_pages, &a.c));
  if (!elem_size(dtype)) return fail(NHIP_STATUS_UNSUPPORTED, "kv8: dtype has to be F32, F16 or BF16");
  if (batch < 0 || tokens < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "kv8: negative extent");
  if (batch == 0 || tokens == 0) return ok();
  if (!key || !value || !starts) return fail(NHIP_STATUS_NULL_POINTER, "kv8: null pointer");
  if (!aligned_to(key, 16) || !aligned_to(value, 16))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "kv8: the values read have to be 16-byte aligned");
  a.out[0] = key;
  a.out[1] = value;
  a.starts = starts;
  a.tokens = tokens;
  const int64_t items = (int64_t)tokens * a.c.kv_heads * (a.c.head_dim / 8);
  if (tokens > (0x7fffffff - kThreads) / a.c.kv_heads / (a.c.head_dim / 8) ||
      batch > 0x7fffffff / ceil_div(items, kThreads))
    return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "kv8: too many tokens in one call");
  a.items = (int32_t)items;
  a.blocks = (int32_t)ceil_div(items, kThreads);
  a.by_vecs = fast_div(a.c.head_dim / 8);
  a.by_heads = fast_div(a.c.kv_heads);
  return NHIP_FOR_ELEM(dtype, T, read_run<T>(a, (uint32_t)batch * a.blocks, as_stream(stream)));
}

}  // extern "C"
