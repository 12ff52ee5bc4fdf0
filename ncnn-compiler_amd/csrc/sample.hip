// The next token of each row of logits: temperature, top-k, top-p, min-p, and a
// draw by a given uniform number.
//
// Tokens of a row stand in one order: larger logits first, of equal ones the
// lower index.  Every filter keeps the first so many of that order, so what is
// kept is all up to one (logit, index) pair, and is found without sorting the
// row.  Weights exp((l - largest) / T) are formed in 64 bits and held as whole
// multiples of 2^-44: their sums are exact and the same in any order, so results
// do not depend on which atomic came first.  What they are compared with, top-p's
// and the uniform number's share of a sum, is rounded to the whole number that
// decides the same, so a token next to a border is on the side where the exact sums
// of these weights put it.  A weight that rounds to 0 is never drawn.
#include <algorithm>

#include "elem.h"

namespace nhip {
namespace {

constexpr int kBins = 1024;    // of weights' exponents, or of keys, or of indices
constexpr int kMostLogits = 1 << 19;  // of a row: as many weights of 2^44 are the most that 64 bits sum
constexpr int kSorted = 1024;  // tokens that are sorted at most
constexpr int kOnce = 128;     // and for all filters at once, rather than about each one's border (a sort of more takes barriers)
constexpr float kRange = 31.5f;  // exp(-31.5) < 2^-45, which rounds to 0

// What the launches before the last one leave of a row.
struct RowParts {
  uint64_t total;        // of all weights
  uint64_t count;        // of tokens listed (an int32 is counted in)
  uint64_t bins[kBins];  // counts, weights, or the sums of sets of vectors
  // where the border was found: its bin, and what comes before that (bin + 1, 0: not found)
  uint64_t before;
  uint64_t found;
};
constexpr int kRowZeros = kBins + 4;  // of 64 bits, to begin with

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int32_t vocab;
  const float* uniform;
  float temperature, top_p, min_p;
  int32_t top_k;
  const float* temperature_each;  // [rows], in place of the single ones
  const int32_t* top_k_each;
  const float* top_p_each;
  const float* min_p_each;
  int32_t* token;
  float* logprob;
  // rows that several workgroups begin: each one's largest key and bound
  int32_t chunks;
  uint2* tops;      // [rows][chunks]
  RowParts* parts;  // [rows]
  uint32_t* lists;  // [rows][kLongList]: indices of tokens that may be kept (only if a row can have a list)
};
constexpr int kLongList = 16384;


// Keys in the order of the values; -0 and 0 are equal.
__device__ __forceinline__ uint32_t key_of(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Key and index as one number, in the order of the tokens (larger first).
__device__ __forceinline__ uint64_t place_of(uint32_t key, int index) { return (uint64_t)key << 32 | (uint32_t)~index; }

// exp((l - top) / T) in units of 2^-44, to the nearest: 2^(y / 64) as 2^n times a
// table's 2^(i / 64) times the Taylor series of e^(f ln 2 / 64) for |f| <= 1/2, whose
// first term left out is 4e-17.  (No infinite top.)
struct Weights {
  double top, rate;     // 64 log2(e) / T
  const double* table;  // [64]
  __device__ __forceinline__ uint64_t operator()(float l) const {
    const double y = fmax(((double)l - top) * rate, -47.0 * 64);
    // the nearest whole number: in the last bits of a sum with 1.5 2^52
    constexpr double whole = 6755399441055744.0;
    const double m = y + whole, f = y - (m - whole);
    const uint32_t i = (uint32_t)__builtin_bit_cast(uint64_t, m);
    constexpr double c = 0.69314718055994530942 / 64;
    double p = c * c * c * c * c / 120;
    p = fma(p, f, c * c * c * c / 24);
    p = fma(p, f, c * c * c / 6);
    p = fma(p, f, c * c / 2);
    p = fma(p, f, c);
    p = fma(p, f, 1.0);
    // 2^(n + 44) as an addition to the exponent; + 2^52: the sum's last 52 bits are the whole number
    const uint64_t t = __builtin_bit_cast(uint64_t, table[i & 63]) + ((uint64_t)((i << 14 & 0xfff00000u) + (44u << 20)) << 32);
    return __builtin_bit_cast(uint64_t, fma(p, __builtin_bit_cast(double, t), 4503599627370496.0)) & ((uint64_t(1) << 52) - 1);
  }
};

__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

// f n, 0 < f < 1, rounded down or up to a whole number: f is 24 bits times a power of 2.
// All lanes have the same, so that the scalar unit does it (0.3 us of a call less).
__device__ __forceinline__ uint64_t share_of(uint64_t n, float f, bool up) {
  n = lane64(n, 0);
  const uint32_t bits = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(uint32_t, f)), exponent = max(bits >> 23, 1u);
  const uint64_t m = (bits & 0x7fffffu) | (bits >> 23 ? 0x800000u : 0u);
  const uint64_t low = n * m, high = __umul64hi(n, m);  // of n m, below 2^88
  const uint32_t shift = 150 - exponent;                // 24 to 149
  if (shift < 64) return (high << (64 - shift) | low >> shift) + (up && low << (64 - shift));
  if (shift == 64) return high + (up && low);
  const uint64_t q = shift < 128 ? high >> (shift - 64) : 0;
  return q + (up && (low || (shift < 128 ? high << (128 - shift) : high)));
}
// The least sum that reaches top-p's share: a token stays if less comes before it (and the first always).
__device__ __forceinline__ uint64_t limit_of(uint64_t total, float top_p) {
  return top_p > 0.f ? max(share_of(total, top_p, true), uint64_t(1)) : 1;
}

// Sums of the lanes up to each, by moves inside the vector unit: within rows of 16
// lanes, then the rows' last lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  return (uint64_t)moved<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 | moved<CTRL, ROWS>((uint32_t)v);
}
template <class N>
__device__ __forceinline__ N wave_scan(N v) {
  v += moved<0x111, 0xf>(v);  // from 1, 2, 4, 8 lanes before
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);  // the last lane of the row before, to rows 1 and 3
  v += moved<0x143, 0xc>(v);  // lane 31, to rows 2 and 3
  return v;
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return lane64(wave_scan(v), 63); }

__device__ __forceinline__ void add_to(uint64_t& bin, uint64_t m) { atomicAdd((unsigned long long*)&bin, (unsigned long long)m); }
__device__ __forceinline__ void count_in(uint64_t& bin) { atomicAdd((uint32_t*)&bin, 1u); }  // below 2^32 of them

// A row in 16-byte vectors from the aligned place at or before its start; what
// lies outside the row is -infinity and is not read.  NaN is -infinity.  A wave has
// a run of them: share `part` of `parts`.
template <class T>
struct Row {
  static constexpr int V = kVec<T>;
  typedef T VT __attribute__((ext_vector_type(V)));
  const T* from;  // aligned
  int shift, vocab, all, begin, end;  // vectors of the row, of the wave
  __device__ __forceinline__ Row(const T* row, int vocab, int part, int parts) : vocab(vocab) {
    shift = (int)(((uintptr_t)row & 15) / sizeof(T));
    from = row - shift;
    all = (int)(((int64_t)vocab + shift + V - 1) / V);
    begin = (int)((int64_t)part * all / parts);
    end = (int)((int64_t)(part + 1) * all / parts);
  }
  __device__ __forceinline__ int first(int vec) const { return vec * V - shift; }
  __device__ __forceinline__ VT load(int vec) const {
    const int i = first(vec);
    VT v;
    if (i >= 0 && i + V <= vocab) {
      v = *reinterpret_cast<const VT*>(from + (int64_t)vec * V);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = i + j >= 0 && i + j < vocab ? from[(int64_t)vec * V + j] : (T)-INFINITY;
    }
    return v;
  }
  // f(value, index) for the wave's tokens, a vector to a lane
  template <class F>
  __device__ __forceinline__ void each(int lane, F f) const {
    constexpr int U = 4;
    for (int c = begin + lane; c - lane < end; c += 64 * U) {
      VT v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * 64 < end) v[u] = load(c + u * 64);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * 64 < end)
#pragma unroll
          for (int j = 0; j < V; ++j) f(fmaxf((float)v[u][j], -INFINITY), first(c + u * 64) + j);
    }
  }
  // The indices of the wave's tokens that reach `least` (of value `last` up to index
  // `last_index`): `reserve` gives the wave room for so many, put(place, index)
  // takes them.  One reservation for U vectors of every lane; a lane goes through
  // the bits that it has set, so that the few cost little (with the values at hand
  // every place was a branch of its own: 64 x 131072 bf16 59 us a call, so 48).
  template <class R, class F>
  __device__ __forceinline__ void each_from(int lane, float least, float last, int last_index, R reserve, F put) const {
    constexpr int U = 8;
    for (int c = begin + lane; c - lane < end; c += 64 * U) {
      VT v[U];
      uint64_t on = 0;  // bit u V + j
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * 64 < end) v[u] = load(c + u * 64);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * 64 < end) {
          uint32_t bits = 0;
#pragma unroll
          for (int j = 0; j < V; ++j) bits |= (float)v[u][j] >= least ? 1u << j : 0;  // (no NaN)
          if (least == last && bits) {
#pragma unroll
            for (int j = 0; j < V; ++j)
              if ((float)v[u][j] == last && first(c + u * 64) + j > last_index) bits &= ~(1u << j);
          }
          on |= (uint64_t)bits << (u * V);
        }
      const int mine = __popcll(on);
      if (!__any(mine)) continue;
      const int upto = (int)wave_scan((uint32_t)mine);
      int at = reserve(__builtin_amdgcn_readlane(upto, 63)) + upto - mine;
      for (; on; on &= on - 1) {
        const int bit = __builtin_ctzll(on);
        put(at++, first(c + bit / V * 64) + bit % V);
      }
    }
  }
  // Weights of a vector's tokens and their sum: vector `lane` of set `set` of 64.
  template <class F>
  __device__ __forceinline__ uint64_t set_sum(int set, int lane, uint64_t (&w)[V], VT& v, F weight) const {
    uint64_t sum = 0;
    const int vec = set * 64 + lane;
    if (vec < all) {
      v = load(vec);
#pragma unroll
      for (int j = 0; j < V; ++j) sum += w[j] = weight(fmaxf((float)v[j], -INFINITY), first(vec) + j);
    }
    return sum;
  }
  __device__ __forceinline__ int sets() const { return (all + 63) / 64; }
  // sets of a bin: a power of two
  __device__ __forceinline__ int set_shift() const {
    int s = 0;
    while ((sets() - 1) >> s >= kBins) ++s;
    return s;
  }
};

// A row's settings.
struct Settings {
  float temperature, top_p, min_p;
  int k;
  __device__ __forceinline__ Settings(const SampleArgs& a, int64_t r) {
    temperature = a.temperature_each ? a.temperature_each[r] : a.temperature;
    top_p = a.top_p_each ? a.top_p_each[r] : a.top_p;
    min_p = a.min_p_each ? a.min_p_each[r] : a.min_p;
    min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
    k = a.top_k_each ? a.top_k_each[r] : a.top_k;
    if (k <= 0 || k > a.vocab) k = a.vocab;
    if (!(temperature > 0.f)) k = 1;
  }
  // few: a bound on the logits finds the first k
  __device__ __forceinline__ bool few(int vocab) const { return k <= kSorted && k < vocab; }
  __device__ __forceinline__ bool unfiltered(int vocab) const { return k == vocab && !(top_p < 1.f) && min_p == 0.f; }
};

// Distances from the largest logit, in halves, so that none overflows: how far
// tokens weigh anything, and how far the histogram for top-p goes at first (the
// tokens past it seldom hold 1 - top_p of all; they are most of a row, and each
// costs an LDS atomic).
struct Distances {
  float half_top, reach, scope;
  __device__ __forceinline__ Distances(float top, const Settings& c) {
    half_top = 0.5f * top;
    reach = fminf(0.5f * kRange * c.temperature, 3.4028235e38f);  // (finite: -infinity stays outside)
    const float near = 6.f - 2.5f * __logf(fmaxf(1.f - c.top_p, 1e-6f));
    scope = c.top_p < 1.f ? fminf(reach, 0.5f * near * c.temperature) : reach;
  }
  __device__ __forceinline__ float below(float l) const { return fmaf(-0.5f, l, half_top); }
  // a logit that no token of weight is below
  __device__ __forceinline__ float least() const { return fmaxf(2.f * (half_top - reach - 1e-6f * (fabsf(half_top) + reach)), -3.4028235e38f); }
  // ... or of bins 0 .. bin of the histogram up to `scope` (the margin: a bin's rounding)
  __device__ __forceinline__ float least_of(int bin, float rate, float scope) const {
    return bin == kBins - 1 ? least() : fmaxf(least(), 2.f * (half_top - (float)(bin + 1) / rate - 1e-6f * (fabsf(half_top) + scope)));
  }
  __device__ __forceinline__ int bin(float l, float rate) const { return (int)fminf(below(l) * rate, (float)(kBins - 1)); }
};

// A bound that at least as many tokens of the wave reach as is its share of the
// first k: by its lanes' largest.
template <class T>
__device__ __forceinline__ uint32_t wave_bound(const Row<T>& row, float mine, int k) {
  if (row.begin >= row.end) return 0xffffffffu;
  const int want = (int)(((int64_t)k * (row.end - row.begin) + row.all - 1) / row.all);
  const uint32_t key = key_of(mine);
  uint32_t bound = 0;
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
    if (__popcll(__ballot(key >= (bound | bit))) >= want) bound |= bit;
  return bound;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

template <int WAVES>
struct SampleLds {
  static constexpr int kList = WAVES > 4 ? 16384 : 4096;  // tokens that LDS holds
  uint64_t list[kList];
  uint64_t sorted[kSorted];
  uint64_t bins[kBins];
  double table[64];
  uint64_t part[WAVES];
  uint32_t keys[WAVES];
  int32_t count, at, index;
  float logit;
  uint64_t total;
};

// list[0 .. n) in falling order, n at most kSorted.  Steps that stay inside 128
// places are a wave's own.
template <int WAVES>
__device__ __forceinline__ void sort_list(uint64_t* list, int n) {
  constexpr int TH = WAVES * 64;
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += TH) list[i] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run <<= 1)
    for (int gap = run >> 1; gap; gap >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += TH) {
        const int a = (i & ~(gap - 1)) << 1 | (i & (gap - 1)), b = a + gap;
        const uint64_t x = list[a], y = list[b];
        if ((x < y) == ((a & run) == 0)) {
          list[a] = y;
          list[b] = x;
        }
      }
      // (the step before or after one of wider gaps reads what other waves wrote)
      if (gap > 64 || (gap == 1 && run >= 128))
        __syncthreads();
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  __syncthreads();
}

// A place to a lane: the sum of the weights of those of `n` lanes that lie before
// it in the order.
__device__ __forceinline__ uint64_t before_me(uint64_t place, uint64_t w, int n) {
  uint64_t sum = 0;
  for (int j = 0; j < n; ++j) {
    const uint64_t q = lane64(place, j), add = lane64(w, j);
    sum += q > place ? add : 0;
  }
  return sum;
}

// The sum over the bins (or any kBins numbers) up to each, in place; returns the
// sum of all.  At most kBins threads, a power of two.
template <int WAVES>
__device__ __forceinline__ uint64_t scan_bins(SampleLds<WAVES>& s, int lane, int wave) {
  constexpr int EACH = kBins / (WAVES * 64);
  uint64_t v[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) v[i] = sum += s.bins[threadIdx.x * EACH + i];
  const uint64_t upto = wave_scan(sum);
  if (lane == 63) s.part[wave] = upto;
  __syncthreads();
  uint64_t before = upto - sum, all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += s.part[w];
    all += s.part[w];
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) s.bins[threadIdx.x * EACH + i] = before + v[i];
  __syncthreads();
  return all;
}

constexpr int kPartWaves = 4;

// The first launch for long rows: the largest logit of a part of a row, and the bound
// on its share of the first k.  Bytes bound it: 256 rows of 50021 fp32 10.4 us (51 MB, 4.9
// TB/s), 64 of 131072 bf16 5.8 (16.8 MB, most of it a launch's start and end).
template <class T>
__global__ __launch_bounds__(kPartWaves * 64) void sample_top_kernel(SampleArgs a) {
  __shared__ uint2 part[kPartWaves];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks;
  const Row<T> row((const T*)a.logits + r * a.stride, a.vocab, chunk * kPartWaves + wave, a.chunks * kPartWaves);
  const Settings c(a, r);
  float mine = -INFINITY;
  row.each(lane, [&](float l, int) { mine = fmaxf(mine, l); });
  const float top = wave_max(mine);
  const uint32_t bound = c.few(a.vocab) && c.k > 1 ? wave_bound(row, mine, c.k) : 0;
  if (lane == 0) part[wave] = make_uint2(key_of(top), bound);
  for (int i = chunk * kPartWaves * 64 + threadIdx.x; i < kRowZeros; i += a.chunks * kPartWaves * 64) (&a.parts[r].total)[i] = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint2 v = part[0];
#pragma unroll
    for (int w = 1; w < kPartWaves; ++w) v = make_uint2(max(v.x, part[w].x), min(v.y, part[w].y));
    a.tops[r * a.chunks + chunk] = v;
  }
}

// Largest key and bound of a row's parts, for every lane.
__device__ __forceinline__ uint2 row_top(const SampleArgs& a, int64_t r, int lane) {
  uint2 v = make_uint2(0, 0xffffffffu);
  for (int i = lane; i < a.chunks; i += 64) {
    const uint2 t = a.tops[r * a.chunks + i];
    v = make_uint2(max(v.x, t.x), min(v.y, t.y));
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) v = make_uint2(max(v.x, (uint32_t)__shfl_xor((int)v.x, o)), min(v.y, (uint32_t)__shfl_xor((int)v.y, o)));
  return v;
}

// A wave's tokens from `least` on into the row's list.
template <class T>
__device__ __forceinline__ void list_tokens(const SampleArgs& a, int64_t r, const Row<T>& row, int lane, float least) {
  uint32_t* list = a.lists + r * kLongList;
  row.each_from(
      lane, least, INFINITY, 0,
      [&](int m) {
        int at = 0;
        if (lane == 0) at = atomicAdd((int*)&a.parts[r].count, m);
        return __builtin_amdgcn_readfirstlane(at);
      },
      [&](int at, int index) {
        if (at < kLongList) list[at] = (uint32_t)index;
      });
}

// The second: of a part of a row the histogram that the row's border is first
// looked for in, or without a filter the sums of its sets; of rows with top-k of few
// the tokens that reach the bound.  The weights' arithmetic in 64 bits and the 64-bit
// LDS atomics bound it (0.85 lanes of a CU a cycle, of 32 bits 1.7: counts have those):
// 256 rows of 50021 fp32 by top-p 0.95 23.6 us, 64 of 131072 bf16, each its own filters, 10.4.
template <class T>
__global__ __launch_bounds__(kPartWaves * 64) void sample_bins_kernel(SampleArgs a) {
  __shared__ uint64_t bins[kBins];
  __shared__ double table[64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks;
  const Settings c(a, r);
  const bool unfiltered = c.unfiltered(a.vocab);
  if (c.k == 1 || (c.k == a.vocab && !(c.top_p < 1.f) && !unfiltered)) return;
  const uint2 keys = row_top(a, r, lane);
  const float top = of_key(keys.x);
  if (!(fabsf(top) < INFINITY)) return;
  const Row<T> row((const T*)a.logits + r * a.stride, a.vocab, chunk * kPartWaves + wave, a.chunks * kPartWaves);
  const Distances d(top, c);
  const Weights weight{(double)top, 64 * 1.4426950408889634074 / (double)c.temperature, table};
  if (c.few(a.vocab)) {
    list_tokens(a, r, row, lane, fmaxf(d.least(), keys.y > key_of(-INFINITY) ? of_key(keys.y) : -INFINITY));
    return;
  }
  if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x / 64);
  if (unfiltered) {
    __syncthreads();
    const int shift = row.set_shift(), sets = row.sets();
    for (int set = chunk * kPartWaves + wave; set < sets; set += a.chunks * kPartWaves) {
      uint64_t w[Row<T>::V];
      typename Row<T>::VT v;
      const uint64_t sum = wave_sum(row.set_sum(set, lane, w, v, [&](float l, int) { return weight(l); }));
      if (lane == 0) add_to(a.parts[r].bins[set >> shift], sum);
    }
    return;
  }
  for (int i = threadIdx.x; i < kBins; i += kPartWaves * 64) bins[i] = 0;
  __syncthreads();
  const float scope = c.k < a.vocab ? d.reach : d.scope, rate = (float)kBins / scope;
  uint64_t sum = 0;
  if (c.k < a.vocab)
    row.each(lane, [&](float l, int) {
      if (d.below(l) <= scope) count_in(bins[d.bin(l, rate)]);
    });
  else
    row.each(lane, [&](float l, int) {
      const uint64_t w = weight(l);
      sum += w;
      if (d.below(l) <= scope) add_to(bins[d.bin(l, rate)], w);
    });
  sum = wave_sum(sum);
  if (lane == 0 && sum) add_to(a.parts[r].total, sum);
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kPartWaves * 64)
    if (bins[i]) add_to(a.parts[r].bins[i], bins[i]);
}

// The third, of rows with a histogram: the bin of the border, and the tokens up to it.
// 64 rows of 131072 bf16 6.2 us: every workgroup sums the histogram before it reads.
template <class T>
__global__ __launch_bounds__(kPartWaves * 64) void sample_list_kernel(SampleArgs a) {
  __shared__ uint64_t part[kPartWaves];
  __shared__ int found;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks;
  const Settings c(a, r);
  if (c.few(a.vocab) || (c.k == a.vocab && !(c.top_p < 1.f))) return;
  const float top = of_key(row_top(a, r, lane).x);
  if (!(fabsf(top) < INFINITY)) return;
  constexpr int EACH = kBins / (kPartWaves * 64);
  uint64_t v[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) v[i] = sum += a.parts[r].bins[threadIdx.x * EACH + i];
  const uint64_t limit = c.k < a.vocab ? (uint64_t)c.k : limit_of(a.parts[r].total, c.top_p);
  const uint64_t upto = wave_scan(sum);
  if (lane == 63) part[wave] = upto;
  if (threadIdx.x == 0) found = -1;
  __syncthreads();
  uint64_t before = upto - sum, all = 0;
#pragma unroll
  for (int w = 0; w < kPartWaves; ++w) {
    if (w < wave) before += part[w];
    all += part[w];
  }
  // (no border: all are kept, or it lies past the histogram)
  if (all < limit || (c.k < a.vocab && all == limit)) return;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const uint64_t ahead = before + (i ? v[i - 1] : 0);
    if (before + v[i] >= limit && ahead < limit) {
      found = threadIdx.x * EACH + i;
      if (chunk == 0) {
        a.parts[r].before = ahead;
        a.parts[r].found = found + 1;
      }
    }
  }
  __syncthreads();
  const Distances d(top, c);
  const float scope = c.k < a.vocab ? d.reach : d.scope;
  const Row<T> row((const T*)a.logits + r * a.stride, a.vocab, chunk * kPartWaves + wave, a.chunks * kPartWaves);
  list_tokens(a, r, row, lane, d.least_of(found, (float)kBins / scope, scope));
}

// One workgroup: one row, or what is left of it to do.
//
// Tokens that may be kept are put together in LDS.  For top-k of few a bound that
// at least k tokens reach, from the lanes' largest ones, leaves a few hundred.
// Otherwise a histogram of the tokens by their weights' exponents, of counts for
// top-k and of weights for top-p, says in which bin the border lies.  The tokens
// about the border are sorted, or if they are too many their bin is divided
// further by the logits' bits, down to equal ones, of which the first by index are
// kept.  The draw sums weights by index: of the tokens in LDS, or, if they do not
// fit there, of all.
//
// A chain of steps between barriers bounds it, of which each has little to do: 64 rows
// of 131072 bf16, each its own filters, 22.4 us behind the launches above; 16 of 1000 fp32 by
// top-k 12.1 a call.  256 of 50021 fp32 by top-p 0.95, all in this launch, 68: the largest,
// the histogram and the tokens that it leaves (some 9000) are a pass over the row each,
// of one CU, and the tokens are summed twice.
template <class T, int WAVES, bool PARTS>
__global__ __launch_bounds__(WAVES * 64) void sample_kernel(SampleArgs a) {
  constexpr int TH = WAVES * 64;
  constexpr int kList = SampleLds<WAVES>::kList;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  SampleLds<WAVES>& s = *reinterpret_cast<SampleLds<WAVES>*>(lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x;
  const Row<T> row((const T*)a.logits + r * a.stride, a.vocab, wave, WAVES);
  const Settings c(a, r);
  const int k = c.k;

  uint32_t top_key = 0, bound = 0xffffffffu;
  if constexpr (PARTS) {
    const uint2 v = row_top(a, r, lane);
    top_key = v.x;
    bound = v.y;
    if (threadIdx.x < 64) s.table[threadIdx.x] = exp2((double)threadIdx.x / 64);
    __syncthreads();
  } else {
    float mine = -INFINITY;
    row.each(lane, [&](float l, int) { mine = fmaxf(mine, l); });
    const float top = wave_max(mine);
    if (c.few(a.vocab) && k > 1) bound = wave_bound(row, mine, k);
    if (lane == 0) {
      s.part[wave] = key_of(top);
      s.keys[wave] = bound;
    }
    if (threadIdx.x < 64) s.table[threadIdx.x] = exp2((double)threadIdx.x / 64);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      top_key = max(top_key, (uint32_t)s.part[w]);
      bound = min(bound, s.keys[w]);
    }
  }
  const float top = of_key(top_key);
  if (top == -INFINITY) {  // no token
    if (threadIdx.x == 0) {
      a.token[r] = -1;
      a.logprob[r] = -INFINITY;
    }
    return;
  }
  const Distances d(top, c);
  const Weights weight{(double)top, 64 * 1.4426950408889634074 / (double)(c.temperature > 0.f ? c.temperature : 1.f), s.table};
  const float u = a.uniform[r];
  // the first whose cumulated weight is past this (NaN: 0)
  const auto target_of = [&](uint64_t total) { return u >= 1.f ? total - 1 : u > 0.f ? share_of(total, u, false) : 0; };
  const auto too_light = [&](uint64_t w) { return (double)w * 0x1p-44 < (double)c.min_p; };
  // one thread has found the token; all call the second
  const auto found = [&](int index, float l, uint64_t total) {
    s.index = index;
    s.logit = l;
    s.total = total;
  };
  const auto finish = [&]() {
    __syncthreads();
    if (threadIdx.x == 0) {
      const double x = s.logit == top ? 0.0 : ((double)s.logit - (double)top) / (double)c.temperature;
      a.token[r] = s.index;
      a.logprob[r] = (float)(x - log((double)s.total * 0x1p-44));
    }
  };
  const auto zero_bins = [&]() {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
    if (threadIdx.x == 0) s.count = s.at = 0;
    __syncthreads();
  };
  // s.at: the first bin of the sums whose sum is past this
  const auto find_bin = [&](uint64_t target) {
    for (int i = threadIdx.x; i < kBins; i += TH)
      if (target < s.bins[i] && target >= (i ? s.bins[i - 1] : 0)) s.at = i;
    __syncthreads();
  };
  // tokens of a value: how many, and (behind that) s.at the index of the `left`-th, from 1
  const auto count_equal = [&](float value) {
    int held = 0;
    row.each(lane, [&](float l, int) { held += l == value; });
    const int of_wave = (int)wave_sum((uint64_t)held);
    __syncthreads();
    if (lane == 0) s.keys[wave] = of_wave;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += s.keys[w];
    return all;
  };
  const auto find_equal = [&](float value, int left) {
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      if (w < wave) left -= (int)s.keys[w];
    if (left > 0 && left <= (int)s.keys[wave]) {
      // this wave has it: a vector to a lane, rising
      for (int v0 = row.begin; v0 < row.end; v0 += 64) {
        int n = 0;
        typename Row<T>::VT v;
        if (v0 + lane < row.end) {
          v = row.load(v0 + lane);
#pragma unroll
          for (int j = 0; j < Row<T>::V; ++j) n += (float)v[j] == value;
        }
        const int upto = (int)wave_scan((uint32_t)n);
        if (upto >= left && upto - n < left) {
          int need = left - (upto - n);
#pragma unroll
          for (int j = 0; j < Row<T>::V; ++j)
            if ((float)v[j] == value && --need == 0) s.at = row.first(v0 + lane) + j;
        }
        const int all_here = __builtin_amdgcn_readlane(upto, 63);
        if (all_here >= left) break;
        left -= all_here;
      }
    }
    __syncthreads();
  };

  if (k == 1) {
    // the lowest index of the largest
    int low = 0x7fffffff;
    row.each(lane, [&](float l, int index) {
      if (l == top) low = min(low, index);
    });
#pragma unroll
    for (int o = 32; o; o >>= 1) low = min(low, __shfl_xor(low, o));
    __syncthreads();
    if (lane == 0) s.keys[wave] = low;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
      for (int w = 1; w < WAVES; ++w) low = min(low, (int)s.keys[w]);
      a.token[r] = low;
      a.logprob[r] = 0.f;
    }
    return;
  }
  if (top == INFINITY) {
    // infinite ones weigh the same, others nothing
    const int64_t all = min(count_equal(top), (int64_t)k);
    const int kept = (int)(c.top_p < 1.f ? limit_of(all, c.top_p) : all);
    const uint64_t total = (uint64_t)kept << 44;
    find_equal(top, (int)(target_of(total) >> 44) + 1);
    if (threadIdx.x == 0) found(s.at, top, total);
    finish();
    return;
  }

  // what is kept: everything up to (last, last_index) of the order, as far as it weighs anything
  float last = -INFINITY;
  int last_index = 0x7fffffff;
  const auto inside = [&](float l, int index) { return d.below(l) <= d.reach && l >= last && (l > last || index <= last_index); };
  const auto inside_place = [&](uint64_t p) { return inside(of_key((uint32_t)(p >> 32)), (int)~(uint32_t)p); };
  // n tokens by their indices into s.list, the values of four of a thread on their way at a time
  int n = 0;
  const auto gather = [&](auto index_of) {
    if (n <= kList)
      for (int i0 = threadIdx.x; i0 < n; i0 += 4 * TH) {
        int index[4];
        float l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          index[e] = i0 + e * TH < n ? (int)index_of(i0 + e * TH) : 0;  // (others' entries may be places already)
          l[e] = (float)row.from[(int64_t)index[e] + row.shift];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i0 + e * TH < n) s.list[i0 + e * TH] = place_of(key_of(l[e]), index[e]);
      }
    __syncthreads();
  };
  // the tokens from `least` on together in LDS; false: they do not fit
  const auto collect = [&](float least) {
    zero_bins();
    row.each_from(
        lane, fmaxf(fmaxf(least, last), d.least()), last, last_index,
        [&](int m) {
          int at = 0;
          if (lane == 0) at = atomicAdd(&s.count, m);
          return __builtin_amdgcn_readfirstlane(at);
        },
        [&](int at, int index) {
          if (at < kList) s.list[at] = (uint32_t)index;
        });
    __syncthreads();
    n = s.count;
    gather([&](int i) { return (uint32_t)s.list[i]; });
    return n <= kList;
  };
  // ... from the row's list, where it was begun by others
  const auto collect_listed = [&]() {
    n = (int)a.parts[r].count;
    const uint32_t* list = a.lists + r * kLongList;
    gather([&](int i) { return list[i]; });
    return n <= kList;
  };
  // s.bins: the sums of `measure` over the first m of s.sorted up to each, and behind them the whole
  const auto sum_sorted = [&](int m, auto measure) {
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = i < m ? measure(s.sorted[i]) : 0;
    __syncthreads();
    return scan_bins(s, lane, wave);
  };
  const auto weight_of = [&](uint64_t place) { return weight(of_key((uint32_t)(place >> 32))); };

  bool listed = false;
  uint64_t mass = 0;  // of all that top-k has left, if top-p's histogram was made
  if (c.few(a.vocab)) {
    const float least = bound > key_of(-INFINITY) ? of_key(bound) : -INFINITY;
    listed = PARTS ? collect_listed() : collect(least);
  }
#pragma unroll 1
  for (int by = 0; by < 2; ++by) {  // top-k by count, then top-p by weight
    if (by == 0 ? k == a.vocab : !(c.top_p < 1.f)) continue;
    if (listed && n <= kOnce) break;  // all in one go, below
    const auto measure = [&](float l) { return by ? weight(l) : (uint64_t)1; };
    float scope = d.reach;
    uint64_t limit;
    uint64_t before = 0;                   // the measure of what comes before the present bin
    uint32_t low = 0, high = 0xffffffffu;  // its keys
    int bin = -1, shift = 0;               // its bin of weights
    const bool begun = PARTS && (by == 0 ? !c.few(a.vocab) : k == a.vocab);
    if (begun && a.parts[r].found) {
      scope = by ? d.scope : d.reach;
      if (by) mass = a.parts[r].total;
      limit = by ? limit_of(mass, c.top_p) : (uint64_t)k;
      before = a.parts[r].before;
      bin = (int)a.parts[r].found - 1;
      listed = collect_listed();
      if (listed && n <= kOnce) break;
    } else {
      for (bool again = false;; again = true) {
        // (with both filters the second looks at what the first has left)
        scope = by && k == a.vocab && !again ? d.scope : d.reach;
        const float rate = (float)kBins / scope;
        uint64_t all;
        zero_bins();
        if (listed) {
          for (int i = threadIdx.x; i < n; i += TH)
            if (const float l = of_key((uint32_t)(s.list[i] >> 32)); inside_place(s.list[i])) add_to(s.bins[d.bin(l, rate)], measure(l));
          __syncthreads();
          all = scan_bins(s, lane, wave);
        } else if (begun && !again) {
          for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = a.parts[r].bins[i];
          __syncthreads();
          all = scan_bins(s, lane, wave);
          if (by) all = a.parts[r].total;
        } else if (by == 0) {
          row.each(lane, [&](float l, int) {
            if (d.below(l) <= scope) count_in(s.bins[d.bin(l, rate)]);
          });
          __syncthreads();
          all = scan_bins(s, lane, wave);
        } else {
          uint64_t sum = 0;
          row.each(lane, [&](float l, int index) {
            const uint64_t w = weight(l);
            if (inside(l, index)) {
              sum += w;
              if (d.below(l) <= scope) add_to(s.bins[d.bin(l, rate)], w);
            }
          });
          sum = wave_sum(sum);
          __syncthreads();
          scan_bins(s, lane, wave);
          if (lane == 0) s.part[wave] = sum;
          __syncthreads();
          all = 0;
#pragma unroll
          for (int w = 0; w < WAVES; ++w) all += s.part[w];
        }
        limit = by ? limit_of(all, c.top_p) : (uint64_t)k;
        if (by) mass = all;
        if (scope == d.reach || s.bins[kBins - 1] >= limit) break;
      }
      // kept: those with less than `limit` before them; the last of them lies in the bin that reaches it
      if (s.bins[kBins - 1] < limit || (by == 0 && s.bins[kBins - 1] == limit)) continue;
    }
    const float rate = (float)kBins / scope;
    for (bool first = bin < 0, again = false;; again = true) {
      if (first || again) {
        // the first bin with which the sum reaches the limit
        __syncthreads();
        if (threadIdx.x == 0) s.at = kBins - 1;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += TH)
          if (before + s.bins[i] >= limit && !(i && before + s.bins[i - 1] >= limit)) s.at = i;
        __syncthreads();
        const int at = s.at;
        before += at ? s.bins[at - 1] : 0;
        if (!again) {
          bin = at;
          // all up to the bin's last value into LDS
          if (!listed) {
            listed = collect(d.least_of(bin, rate, scope));
            if (listed && n <= kOnce) break;
          }
        } else {  // bins of keys: the largest first
          const uint32_t width = 1u << shift;
          high -= (uint32_t)at * width;
          low = high - low >= width ? high - (width - 1) : low;
        }
      }
      __syncthreads();
      if (threadIdx.x == 0) s.count = 0;
      __syncthreads();
      const auto here = [&](float l, int index) {
        if (!inside(l, index) || d.below(l) > scope || d.bin(l, rate) != bin) return false;
        const uint32_t key = key_of(l);
        return key >= low && key <= high;
      };
      uint32_t most = 0, least = 0xffffffffu;
      const auto take = [&](float l, int index) {
        if (here(l, index)) {
          const uint32_t key = key_of(l);
          most = max(most, key);
          least = min(least, key);
          const int i = atomicAdd(&s.count, 1);
          if (i < kSorted) s.sorted[i] = place_of(key, index);
        }
      };
      if (listed)
        for (int i = threadIdx.x; i < n; i += TH) take(of_key((uint32_t)(s.list[i] >> 32)), (int)~(uint32_t)s.list[i]);
      else
        row.each(lane, take);
#pragma unroll
      for (int o = 32; o; o >>= 1) {
        most = max(most, (uint32_t)__shfl_xor((int)most, o));
        least = min(least, (uint32_t)__shfl_xor((int)least, o));
      }
      if (lane == 0) s.part[wave] = (uint64_t)most << 32 | least;
      __syncthreads();
      const int count = s.count;
      if (count <= 64) {
        if (wave == 0) {
          const uint64_t place = lane < count ? s.sorted[lane] : 0;
          const uint64_t m = lane < count ? measure(of_key((uint32_t)(place >> 32))) : 0;
          const uint64_t ahead = before_me(place, m, count);
          // the last of those that stay has the most before it
          const bool stays = m && before + ahead < limit;
          if (lane == 0) s.total = 0;
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          if (stays) atomicMax((unsigned long long*)&s.total, (unsigned long long)ahead + 1);
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          if (stays && ahead + 1 == *(volatile uint64_t*)&s.total) s.part[0] = place;
        }
        __syncthreads();
        last = of_key((uint32_t)(s.part[0] >> 32));
        last_index = (int)~(uint32_t)s.part[0];
        __syncthreads();
        break;
      }
      if (count <= kSorted) {
        sort_list<WAVES>(s.sorted, count);
        sum_sorted(count, [&](uint64_t place) { return measure(of_key((uint32_t)(place >> 32))); });
        if (threadIdx.x == 0) s.at = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += TH)
          if (before + (i ? s.bins[i - 1] : 0) < limit) atomicMax(&s.at, i);
        __syncthreads();
        const uint64_t place = s.sorted[s.at];
        last = of_key((uint32_t)(place >> 32));
        last_index = (int)~(uint32_t)place;
        __syncthreads();
        break;
      }
      low = 0xffffffffu;
      high = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        high = max(high, (uint32_t)(s.part[w] >> 32));
        low = min(low, (uint32_t)s.part[w]);
      }
      __syncthreads();
      if (low == high) {
        // one value: the first so many by index (of those that top-k has left)
        const float value = of_key(low);
        const uint64_t each = max(measure(value), uint64_t(1));
        const int keep = (int)min((limit - before + each - 1) / each, (uint64_t)count);
        count_equal(value);
        find_equal(value, keep);
        last = value;
        last_index = s.at;
        break;
      }
      // the bin's keys, largest first, into kBins parts
      shift = 0;
      while (((high - low) >> shift) >= (uint32_t)kBins) ++shift;
      zero_bins();
      const auto divide = [&](float l, int index) {
        if (here(l, index)) add_to(s.bins[(high - key_of(l)) >> shift], measure(l));
      };
      if (listed)
        for (int i = threadIdx.x; i < n; i += TH) divide(of_key((uint32_t)(s.list[i] >> 32)), (int)~(uint32_t)s.list[i]);
      else
        row.each(lane, divide);
      __syncthreads();
      scan_bins(s, lane, wave);
    }
    if (listed && n <= kOnce) break;
  }

  if (listed && n <= kOnce) {
    // ------------------------- all that may be kept, sorted: every filter at once (a listed
    // token may lie outside, by the margin of `least`, and takes no place in the order)
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += TH) s.sorted[i] = inside_place(s.list[i]) ? s.list[i] : 0;
    __syncthreads();
    sort_list<WAVES>(s.sorted, n);
    const int first = min(n, k);
    const uint64_t sum = sum_sorted(first, weight_of);
    if (!mass) mass = sum;  // (the list holds the first k)
    const uint64_t limit = c.top_p < 1.f ? limit_of(mass, c.top_p) : ~uint64_t(0);
    if (threadIdx.x == 0) s.at = 1;
    __syncthreads();
    for (int i = threadIdx.x; i < first; i += TH) {
      const uint64_t before = i ? s.bins[i - 1] : 0;
      if (s.bins[i] != before && before < limit && !too_light(s.bins[i] - before)) atomicMax(&s.at, i + 1);
    }
    __syncthreads();
    const uint64_t place = s.sorted[s.at - 1];
    last = of_key((uint32_t)(place >> 32));
    last_index = (int)~(uint32_t)place;
  } else if (!listed && c.min_p > 0.f) {
    // a logit below this is too light (to a margin: its weight decides)
    const float cut = (float)((double)top + (double)c.temperature * (log((double)c.min_p) - 1e-6) - 1e-6 * fabs((double)top));
    listed = collect(fmaxf(last, cut));
  } else if (!listed && last > -INFINITY) {
    listed = collect(last);
  }

  // the draw: weights by index
  if (listed) {
    static_assert(kMostLogits / kBins <= kSorted, "a bin of indices fits s.sorted");
    int shift = 0;
    while ((a.vocab - 1) >> shift >= kBins) ++shift;
    const auto drawn = [&](uint64_t place) -> uint64_t {
      if (!inside_place(place)) return 0;
      const uint64_t w = weight_of(place);
      return too_light(w) ? 0 : w;
    };
    zero_bins();
    for (int i = threadIdx.x; i < n; i += TH)
      if (const uint64_t w = drawn(s.list[i])) add_to(s.bins[~(uint32_t)s.list[i] >> shift], w);
    __syncthreads();
    const uint64_t total = scan_bins(s, lane, wave), target = target_of(total);
    find_bin(target);
    const int at = s.at;
    const uint64_t begin = at ? s.bins[at - 1] : 0;
    for (int i = threadIdx.x; i < n; i += TH)
      if ((int)(~(uint32_t)s.list[i] >> shift) == at && drawn(s.list[i])) {
        // (the index turned round: falling order is rising index)
        s.sorted[atomicAdd(&s.count, 1)] = s.list[i] << 32 | s.list[i] >> 32;
      }
    __syncthreads();
    const int m = s.count;
    if (m <= 64) {
      if (wave == 0) {
        const uint64_t place = lane < m ? s.sorted[lane] : 0, w = lane < m ? weight(of_key((uint32_t)place)) : 0;
        const uint64_t from = before_me(place, w, m), rest = target - begin;
        if (lane < m && rest >= from && rest < from + w) found((int)~(uint32_t)(place >> 32), of_key((uint32_t)place), total);
      }
      finish();
      return;
    }
    sort_list<WAVES>(s.sorted, m);
    sum_sorted(m, [&](uint64_t place) { return weight(of_key((uint32_t)place)); });
    const uint64_t rest = target - begin;
    for (int i = threadIdx.x; i < m; i += TH)
      if (rest < s.bins[i] && rest >= (i ? s.bins[i - 1] : 0)) found((int)~(uint32_t)(s.sorted[i] >> 32), of_key((uint32_t)s.sorted[i]), total);
    finish();
    return;
  }
  const auto drawn = [&](float l, int index) -> uint64_t {
    if (!inside(l, index)) return 0;
    const uint64_t w = weight(l);
    return too_light(w) ? 0 : w;
  };
  const int set_shift = row.set_shift(), sets = row.sets();
  zero_bins();
  if (PARTS && c.unfiltered(a.vocab)) {
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = a.parts[r].bins[i];
  } else {
#pragma unroll 1
    for (int set = wave; set < sets; set += WAVES) {
      uint64_t w[Row<T>::V];
      typename Row<T>::VT v;
      const uint64_t sum = wave_sum(row.set_sum(set, lane, w, v, drawn));
      if (lane == 0) add_to(s.bins[set >> set_shift], sum);
    }
  }
  __syncthreads();
  const uint64_t total = scan_bins(s, lane, wave), target = target_of(total);
  find_bin(target);
  if (wave == 0) {
    const int at = s.at;
    uint64_t begin = at ? s.bins[at - 1] : 0;
    for (int set = at << set_shift; set < min(sets, (at + 1) << set_shift); ++set) {
      uint64_t w[Row<T>::V];
      typename Row<T>::VT v;
      const uint64_t sum = row.set_sum(set, lane, w, v, drawn), upto = wave_scan(sum), all = lane64(upto, 63);
      if (target < begin + all) {
        uint64_t from = begin + upto - sum;
        if (target >= from && target < from + sum) {
#pragma unroll
          for (int j = 0; j < Row<T>::V; ++j) {
            if (target >= from && target < from + w[j]) found(row.first(set * 64 + lane) + j, fmaxf((float)v[j], -INFINITY), total);
            from += w[j];
          }
        }
        break;
      }
      begin += all;
    }
  }
  finish();
}

// What of a filter all rows surely leave out.
bool no_top_k(const nhip_sample_desc* d) { return !d->top_k_each && (d->top_k == 0 || d->top_k >= d->vocab); }
bool no_top_p(const nhip_sample_desc* d) { return !d->top_p_each && d->top_p >= 1.f; }
bool no_filter(const nhip_sample_desc* d) { return no_top_k(d) && no_top_p(d) && !d->min_p_each && d->min_p == 0.f; }
// Rows of which the largest alone counts, or all that min-p leaves, have neither a histogram nor a list.
bool greedy(const nhip_sample_desc* d) {
  return (!d->temperature_each && d->temperature == 0.f) || (!d->top_k_each && d->top_k == 1);
}
bool has_lists(const nhip_sample_desc* d) { return !greedy(d) && !(no_top_k(d) && no_top_p(d)); }
bool has_bins(const nhip_sample_desc* d) { return !greedy(d) && (has_lists(d) || no_filter(d)); }

// Workgroups that begin a row, 0: one does all of it.  They save of its passes over
// the row what the other CUs can take, and cost two or three launches.  us a call, one /
// several, rows x logits fp32 (bf16 alike but for 128 rows and more, which it reads faster):
//            top-p 0.9           no filter           top-k of 3000       top-k of 50
//           32768 65536 131072   32768 65536 131072  65536    131072     65536     131072
//     1     28/23 46/27 80/34    22/17 38/17 68/17   32/29    53/37      24/25     31/28
//    64     32/35 49/41 88/56    23/18 38/21 69/28   39/44    55/53      25/28     34/32
//   128     32/39 51/51 107/86   23/21 39/29 79/45   40/54    73/77      26/31     45/48
//   256     32/44 72/77 133/128  23/28 50/45 87/70   67/78   100/108     42/48     64/62
// The largest alone (16 x 131072, three tensors in turn) 20.6 / 20.1.
int chunks_of(const nhip_sample_desc* d) {
  const int force = setting_int("NHIP_SAMPLE_CHUNKS", -1);
  if (force >= 0) return std::min(force, 64);
  if (!d->temperature_each && d->temperature == 0.f) return 0;
  const double cus = cu_count(), rows = std::max(d->rows, 1);
  double per, cost, share = 1 - rows / cus;  // ns of a logit, us, of the passes
  if (no_filter(d)) {
    per = 0.38, cost = 8, share = std::max(0.5, 1 - rows / (2 * cus));  // (the last launch reads few)
  } else if (!d->top_k_each && d->top_k > 0 && d->top_k < d->vocab) {
    per = d->top_k <= kSorted ? 0.05 : 0.13, cost = d->top_k <= kSorted ? 6 : 9;
  } else if (no_top_p(d) && no_top_k(d)) {  // min-p alone: as of few
    per = 0.05, cost = 6;
  } else {
    per = 0.35, cost = 9;
  }
  if (per * 1e-3 * d->vocab * share < cost) return 0;
  const int64_t want = ceil_div(4 * cu_count(), std::max(d->rows, 1));
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, d->vocab / 2048, 64}));
}

uint64_t workspace_of(const nhip_sample_desc* d) {
  const int chunks = chunks_of(d);
  const uint64_t list = has_lists(d) ? kLongList * sizeof(uint32_t) : 0;
  return chunks ? d->rows * (sizeof(RowParts) + (uint64_t)chunks * sizeof(uint2) + list) : 0;
}

template <class T, int WAVES, bool PARTS>
int sample_last(const SampleArgs& a, int rows, hipStream_t s) {
  constexpr int bytes = (int)sizeof(SampleLds<WAVES>);
  if (bytes > 65536) NHIP_TRY(ensure_dynamic_lds((const void*)sample_kernel<T, WAVES, PARTS>, bytes));
  NHIP_LAUNCH("sample", (sample_kernel<T, WAVES, PARTS>), dim3((uint32_t)rows), dim3(WAVES * 64), bytes, s, a);
  return check_launch("sample");
}

template <class T>
int sample_run(const SampleArgs& a, const nhip_sample_desc* d, hipStream_t s) {
  const int rows = d->rows;
  // 16 waves a row, one row a CU, or 4, three a CU, where barriers cost more than the
  // passes or the rows are more than the CUs.  us, 4 / 16: 16 rows of 4096 fp32 by top-k of
  // 50 16.7 / 19.5, of 3000 21.5 / 17.7, top-p 0.9 20.5 / 22.4; of 16384 20.8 / 20.0, 36.6 / 27,
  // 32.4 / 26.1; 1024 of 16384 51 / 83, 81 / 98, 73 / 97, of 32768 bf16 53 / 86, 95 / 124, 101 /
  // 131; past that what top-p keeps seldom fits their part of LDS (512 of 131072 419 / 200).
  if (!a.chunks)
    return a.vocab <= (rows > cu_count() ? 32768 : 8192) ? sample_last<T, 4, false>(a, rows, s) : sample_last<T, 16, false>(a, rows, s);
  const dim3 grid((uint32_t)((int64_t)rows * a.chunks)), block(kPartWaves * 64);
  NHIP_LAUNCH("sample_top", (sample_top_kernel<T>), grid, block, 0, s, a);
  NHIP_TRY(check_launch("sample_top"));
  if (has_bins(d)) {
    NHIP_LAUNCH("sample_bins", (sample_bins_kernel<T>), grid, block, 0, s, a);
    NHIP_TRY(check_launch("sample_bins"));
  }
  if (no_filter(d)) return sample_last<T, 4, true>(a, rows, s);  // (reads a 1024th of a row)
  // (no launch where the settings of all rows leave it nothing to do, nor where the
  // last launch has a workgroup for every CU to do it with: 64 rows of 131072 bf16, each
  // its own settings 50 us without, 45 with; 256 of 50021 fp32 74 and 79)
  const bool some_k = a.top_k_each || a.top_k == 0 || a.top_k > kSorted, some_p = !no_top_p(d);
  const bool many_k = a.top_k_each || (a.top_k > kSorted && a.top_k < a.vocab);
  if (rows <= cu_count() / 2 && (a.temperature_each || a.temperature > 0.f) && some_k && (some_p || many_k)) {
    NHIP_LAUNCH("sample_list", (sample_list_kernel<T>), grid, block, 0, s, a);
    NHIP_TRY(check_launch("sample_list"));
  }
  return sample_last<T, 16, true>(a, rows, s);
}

int sample_args(const nhip_sample_desc* d) {
  if (!d) return fail(NHIP_STATUS_NULL_POINTER, "sample: null descriptor");
  if (!elem_size(d->dtype)) return fail(NHIP_STATUS_UNSUPPORTED, "sample: dtype has to be F32, F16 or BF16");
  if (d->rows < 0 || d->vocab <= 0) return fail(NHIP_STATUS_INVALID_SHAPE, "sample: a row holds at least one logit");
  // (a launch has below 2^32 threads)
  if (d->vocab > kMostLogits || d->rows >= 1 << 22) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "sample: below 2^22 rows of at most 2^19 logits");
  if (d->row_stride < 0) return fail(NHIP_STATUS_INVALID_SHAPE, "sample: negative stride");
  // (values that a tensor holds for each row are read on the device, where these mean the same as the nearest that is allowed)
  if (!(d->temperature >= 0.f) || d->top_k < 0 || !(d->top_p >= 0.f) || !(d->min_p >= 0.f) || d->min_p > 1.f)
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "sample: temperature, top_k and top_p are not negative, min_p 0 to 1");
  if (!aligned_to(d->temperature_each, 4) || !aligned_to(d->top_k_each, 4) || !aligned_to(d->top_p_each, 4) ||
      !aligned_to(d->min_p_each, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "sample: a tensor is not aligned to its type");
  return ok();
}

}  // namespace
}  // namespace nhip

using namespace nhip;

extern "C" {

int nhip_sample_workspace_size(const nhip_sample_desc* desc, uint64_t* bytes) {
  if (!bytes) return fail(NHIP_STATUS_NULL_POINTER, "sample: null pointer");
  NHIP_TRY(sample_args(desc));
  *bytes = workspace_of(desc);
  return ok();
}

int nhip_sample_forward(const nhip_sample_desc* desc, const void* logits, const float* uniform, int32_t* token,
                        float* logprob, void* workspace, uint64_t workspace_bytes, void* stream) {
  NHIP_TRY(sample_args(desc));
  if (desc->rows == 0) return ok();
  if (!logits || !uniform || !token || !logprob) return fail(NHIP_STATUS_NULL_POINTER, "sample: null pointer");
  if (!aligned_to(logits, elem_size(desc->dtype)) || !aligned_to(uniform, 4) || !aligned_to(token, 4) || !aligned_to(logprob, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "sample: a tensor is not aligned to its type");
  const uint64_t need = workspace_of(desc);
  if (need && !workspace) return fail(NHIP_STATUS_NULL_POINTER, "sample: null workspace");
  if (need && (workspace_bytes < need || !aligned_to(workspace, 16)))
    return fail(NHIP_STATUS_OUTPUT_CAPACITY_INSUFFICIENT, "sample: workspace too small or not 16-byte aligned");
  RowParts* parts = (RowParts*)workspace;
  uint2* tops = (uint2*)(parts + desc->rows);
  const SampleArgs a{logits,           desc->row_stride,       desc->vocab,      uniform,          desc->temperature,
                     desc->top_p,      desc->min_p,            desc->top_k,      desc->temperature_each,
                     desc->top_k_each, desc->top_p_each,       desc->min_p_each, token,            logprob,
                     chunks_of(desc),  tops, parts, has_lists(desc) ? (uint32_t*)(tops + (int64_t)desc->rows * chunks_of(desc)) : nullptr};
  return NHIP_FOR_ELEM(desc->dtype, T, sample_run<T>(a, desc, as_stream(stream)));
}

}  // extern "C"
