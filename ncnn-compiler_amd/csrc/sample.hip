// The next token of each row of logits: temperature, top-k, top-p, min-p, and a
// draw by a given uniform number.
//
// Tokens of a row stand in one order: larger logits first, of equal ones the
// lower index.  Every filter keeps the first so many of that order, so what is
// kept is all up to one (logit, index) pair, and is found without sorting the
// row.  Weights exp((l - largest) / T) are formed in 64 bits and held as whole
// multiples of 2^-44: their sums are exact and the same in any order, so results
// do not depend on which atomic came first, and a token next to a border is on
// the side where the exact sums put it (but for those 2^-45).  A weight that
// rounds to 0 is never drawn.
#include <algorithm>

#include "elem.h"

namespace nhip {
namespace {

constexpr int kBins = 1024;   // of weights' exponents, or of keys, or of indices
constexpr int kSorted = 1024;  // tokens that are sorted
constexpr int kList = 4096;   // tokens that LDS holds
constexpr float kRange = 31.5f;  // exp(-31.5) < 2^-45, which rounds to 0

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
};

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

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) {
  return (uint64_t)__shfl_xor((uint32_t)(v >> 32), o) << 32 | __shfl_xor((uint32_t)v, o);
}
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += shfl_xor64(v, o);
  return v;
}
// Sum of the lanes up to this one.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint64_t u = (uint64_t)__shfl_up((uint32_t)(v >> 32), o) << 32 | __shfl_up((uint32_t)v, o);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}

__device__ __forceinline__ void add_to(uint64_t& bin, uint64_t m) { atomicAdd((unsigned long long*)&bin, (unsigned long long)m); }
__device__ __forceinline__ void count_in(uint64_t& bin) { atomicAdd((uint32_t*)&bin, 1u); }  // below 2^32 of them

// A row in 16-byte vectors from the aligned place at or before its start, dealt
// to the waves in runs; what lies outside the row is -infinity and is not read.
// NaN is -infinity.
template <class T, int WAVES>
struct Row {
  static constexpr int V = kVec<T>;
  typedef T VT __attribute__((ext_vector_type(V)));
  const T* from;  // aligned
  int shift, vocab, all, begin, end;  // vectors of the row, the wave's
  __device__ __forceinline__ Row(const T* row, int vocab, int wave) : vocab(vocab) {
    shift = (int)(((uintptr_t)row & 15) / sizeof(T));
    from = row - shift;
    all = (int)(((int64_t)vocab + shift + V - 1) / V);
    begin = (int)((int64_t)wave * all / WAVES);
    end = (int)((int64_t)(wave + 1) * all / WAVES);
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
};

template <int WAVES>
struct SampleLds {
  uint64_t list[kList];
  uint64_t bins[kBins];
  double table[64];
  uint64_t part[WAVES];
  uint32_t keys[WAVES];
  int32_t count, at;
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

// The sum over the bins (or any kBins numbers) up to each, in place; returns the
// sum of all.  At most kBins threads, a power of two.
template <int WAVES>
__device__ __forceinline__ uint64_t scan_bins(SampleLds<WAVES>& s, int lane, int wave) {
  constexpr int EACH = kBins / (WAVES * 64);
  uint64_t v[EACH], sum = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) v[i] = sum += s.bins[threadIdx.x * EACH + i];
  const uint64_t upto = wave_scan(sum, lane);
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

// One workgroup: one row.
//
// top-k of few: a bound that at least k tokens reach, from the lanes' largest
// ones, leaves a few hundred, which are compared with each other.  Otherwise a
// histogram of the tokens by their weights' exponents, of counts for top-k and of
// weights for top-p, says in which bin the border lies; its tokens are compared
// with each other, or if they are too many the bin is divided further by the
// logits' bits, down to equal ones, of which the first by index are kept.
// The draw sums the weights by index: of the kept tokens, put together in LDS, or
// if they are too many, of all.
template <class T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void sample_kernel(SampleArgs a) {
  constexpr int TH = WAVES * 64;
  __shared__ SampleLds<WAVES> s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t r = blockIdx.x;
  const Row<T, WAVES> row((const T*)a.logits + r * a.stride, a.vocab, wave);
  const float temperature = a.temperature_each ? a.temperature_each[r] : a.temperature;
  const float top_p = a.top_p_each ? a.top_p_each[r] : a.top_p;
  float min_p = a.min_p_each ? a.min_p_each[r] : a.min_p;
  min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
  int k = a.top_k_each ? a.top_k_each[r] : a.top_k;
  if (k <= 0 || k > a.vocab) k = a.vocab;
  if (!(temperature > 0.f)) k = 1;

  float mine = -INFINITY;
  row.each(lane, [&](float l, int) { mine = fmaxf(mine, l); });
  float top = mine;
#pragma unroll
  for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  // A bound that at least k tokens reach: of each wave, as many as its share of the
  // row, by its lanes' largest.
  uint32_t bound = 0xffffffffu;
  const bool few = k <= kSorted && k < a.vocab;
  if (few && k > 1 && row.begin < row.end) {
    const int want = (int)(((int64_t)k * (row.end - row.begin) + row.all - 1) / row.all);
    const uint32_t key = key_of(mine);
    bound = 0;
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
      if (__popcll(__ballot(key >= (bound | bit))) >= want) bound |= bit;
  }
  if (lane == 0) {
    s.part[wave] = key_of(top);
    s.keys[wave] = bound;
  }
  if (threadIdx.x == 0) s.count = 0;
  if (threadIdx.x < 64) s.table[threadIdx.x] = exp2((double)threadIdx.x / 64);
  __syncthreads();
  uint32_t top_key = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    top_key = max(top_key, (uint32_t)s.part[w]);
    bound = min(bound, s.keys[w]);
  }
  top = of_key(top_key);
  if (top == -INFINITY) {  // no token
    if (threadIdx.x == 0) {
      a.token[r] = -1;
      a.logprob[r] = -INFINITY;
    }
    return;
  }
  // (of an infinite largest one: 0 where it stands, others as far below as there is)
  const bool infinite = top == INFINITY;
  const Weights exact{infinite ? 0.0 : (double)top, 64 * 1.4426950408889634074 / (double)(temperature > 0.f ? temperature : 1.f), s.table};
  const auto weight = [&](float l) { return exact(infinite ? (l == top ? 0.f : -INFINITY) : l); };
  // half a logit's distance from the largest, and how far tokens weigh anything (halves, so that no difference overflows)
  const float half_top = 0.5f * top, half_reach = fminf(0.5f * kRange * temperature, 3.4e38f);
  const auto below = [&](float l) { return l == top ? 0.f : fmaf(-0.5f, l, half_top); };
  const double u = fmin(fmax((double)a.uniform[r], 0.0), 1.0 - 0x1p-53);  // NaN: 0
  const auto finish = [&](int index, float l, uint64_t total) {
    const double x = l == top ? 0.0 : ((double)l - (double)top) / (double)temperature;
    a.token[r] = index;
    a.logprob[r] = (float)(x - log((double)total * 0x1p-44));
  };
  // the first whose cumulated weight is past this
  const auto target_of = [&](uint64_t total) { return min((uint64_t)((double)total * u), total - 1); };
  // s.bins: the sums of `measure` over the first n <= kSorted of s.list up to each, and behind them the whole
  const auto sum_list = [&](int n, auto measure) {
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = i < n ? measure(of_key((uint32_t)(s.list[i] >> 32))) : 0;
    __syncthreads();
    scan_bins(s, lane, wave);
  };
  // the one of the first n of s.list that is drawn, the weights before it being `begin` and all `total`
  const auto draw_list = [&](int n, uint64_t begin, uint64_t total) {
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += TH) s.list[i] = s.list[i] << 32 | s.list[i] >> 32;  // ~index falls: rising indices
    __syncthreads();
    sort_list<WAVES>(s.list, n);
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = i < n ? weight(of_key((uint32_t)s.list[i])) : 0;
    __syncthreads();
    scan_bins(s, lane, wave);
    const uint64_t target = target_of(total) - begin;
    for (int i = threadIdx.x; i < n; i += TH)
      if (target < s.bins[i] && target >= (i ? s.bins[i - 1] : 0)) finish((int)~(uint32_t)(s.list[i] >> 32), of_key((uint32_t)s.list[i]), total);
  };
  const auto too_light = [&](uint64_t w) { return (double)w * 0x1p-44 < (double)min_p; };

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
      finish(low, top, uint64_t(1) << 44);
    }
    return;
  }
  if (few) {
    // ------------------------------------------------ few tokens are kept
    const float least = bound > key_of(-INFINITY) ? of_key(bound) : -INFINITY;
    row.each(lane, [&](float l, int index) {
      if (l >= least && below(l) <= half_reach) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kSorted) s.list[at] = place_of(key_of(l), index);
      }
    });
    __syncthreads();
    int n = s.count;
    if (n <= kSorted) {
      sort_list<WAVES>(s.list, n);
      n = min(n, k);
      sum_list(n, weight);
      // (the first one always)
      const double limit = top_p < 1.f ? fmax((double)top_p * (double)s.bins[kBins - 1], 1.0) : INFINITY;
      if (threadIdx.x == 0) s.at = 1;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += TH) {
        const uint64_t before = i ? s.bins[i - 1] : 0;
        if ((double)before < limit && !too_light(s.bins[i] - before)) atomicMax(&s.at, i + 1);
      }
      __syncthreads();
      n = s.at;
      draw_list(n, 0, s.bins[n - 1]);
      return;
    }
  }

  // --------------------------------------------------- any number is kept
  // everything up to (last, last_index) of the order, as far as it weighs anything
  float last = -INFINITY;
  int last_index = 0x7fffffff;
  const float rate = (float)kBins / half_reach;
  const auto bin_of = [&](float l) { return (int)fminf(below(l) * rate, (float)(kBins - 1)); };
  const auto inside = [&](float l, int index) { return below(l) <= half_reach && (l > last || (l == last && index <= last_index)); };
#pragma unroll 1
  for (int by = 0; by < 2; ++by) {  // top-k by count, then top-p by weight
    if (by == 0 ? k == a.vocab : !(top_p < 1.f)) continue;
    const auto measure = [&](float l) { return by ? weight(l) : (uint64_t)1; };
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
    __syncthreads();
    row.each(lane, [&](float l, int index) {
      if (inside(l, index))
        by ? add_to(s.bins[bin_of(l)], weight(l)) : count_in(s.bins[bin_of(l)]);
    });
    __syncthreads();
    const uint64_t all = scan_bins(s, lane, wave);
    const double limit = by ? fmax((double)top_p * (double)all, 1.0) : (double)k;  // (the first one always)
    // kept: those with less than `limit` before them; the last of them lies in the bin that reaches it
    if ((double)all < limit || (by == 0 && all <= (uint64_t)k)) continue;
    uint64_t before = 0;                   // the measure of what comes before the present bin
    uint32_t low = 0, high = 0xffffffffu;  // its keys
    int bin = -1, shift = 0;               // its bin of weights
    for (;;) {
      // the first bin with which the sum reaches the limit
      if (threadIdx.x == 0) {
        s.at = kBins - 1;
        s.count = 0;
      }
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += TH)
        if ((double)(before + s.bins[i]) >= limit && s.bins[i]) atomicMin(&s.at, i);
      __syncthreads();
      const int at = s.at;
      if (bin < 0) {
        bin = at;
      } else {  // bins of keys: the largest first
        const uint32_t width = 1u << shift;
        high -= (uint32_t)at * width;
        low = high - low >= width ? high - (width - 1) : low;
      }
      before += at ? s.bins[at - 1] : 0;
      const auto here = [&](float l, int index) {
        if (!inside(l, index) || bin_of(l) != bin) return false;
        const uint32_t key = key_of(l);
        return key >= low && key <= high;
      };
      uint32_t most = 0, least = 0xffffffffu;
      row.each(lane, [&](float l, int index) {
        if (here(l, index)) {
          const uint32_t key = key_of(l);
          most = max(most, key);
          least = min(least, key);
          const int i = atomicAdd(&s.count, 1);
          if (i < kSorted) s.list[i] = place_of(key, index);
        }
      });
#pragma unroll
      for (int o = 32; o; o >>= 1) {
        most = max(most, (uint32_t)__shfl_xor(most, o));
        least = min(least, (uint32_t)__shfl_xor(least, o));
      }
      if (lane == 0) s.part[wave] = (uint64_t)most << 32 | least;
      __syncthreads();
      const int count = s.count;
      if (count <= kSorted) {
        sort_list<WAVES>(s.list, count);
        sum_list(count, measure);
        if (threadIdx.x == 0) s.at = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += TH)
          if ((double)(before + (i ? s.bins[i - 1] : 0)) < limit) atomicMax(&s.at, i);
        __syncthreads();
        const uint64_t place = s.list[s.at];
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
        // one value: the first so many by index
        const float value = of_key(low);
        const int keep = (int)fmax(1.0, fmin(ceil((limit - (double)before) / (double)measure(value)), (double)count));
        int held = 0;
        row.each(lane, [&](float l, int index) { held += l == value && inside(l, index); });
        const uint64_t wave_held = wave_sum((uint64_t)held);
        if (lane == 0) s.part[wave] = wave_held;
        __syncthreads();
        int left = keep;
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
          if (w < wave) left -= (int)s.part[w];
        if (left > 0 && left <= (int)wave_held) {
          // this wave has the last of them: a vector to a lane, rising
          for (int c = row.begin; c < row.end; c += 64) {
            int n = 0;
            typename Row<T, WAVES>::VT v;
            if (c + lane < row.end) {
              v = row.load(c + lane);
#pragma unroll
              for (int j = 0; j < Row<T, WAVES>::V; ++j)
                n += (float)v[j] == value && inside((float)v[j], row.first(c + lane) + j);
            }
            const int upto = (int)wave_scan((uint64_t)n, lane);
            if (upto >= left && upto - n < left) {
              int need = left - (upto - n);
#pragma unroll
              for (int j = 0; j < Row<T, WAVES>::V; ++j)
                if ((float)v[j] == value && inside((float)v[j], row.first(c + lane) + j) && --need == 0) s.at = row.first(c + lane) + j;
            }
            const int all_here = __builtin_amdgcn_readlane(upto, 63);
            if (all_here >= left) break;
            left -= all_here;
          }
        }
        __syncthreads();
        last = value;
        last_index = s.at;
        break;
      }
      // the bin's keys, largest first, into kBins parts
      shift = 0;
      while (((high - low) >> shift) >= (uint32_t)kBins) ++shift;
      for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
      __syncthreads();
      row.each(lane, [&](float l, int index) {
        if (here(l, index))
          by ? add_to(s.bins[(high - key_of(l)) >> shift], weight(l)) : count_in(s.bins[(high - key_of(l)) >> shift]);
      });
      __syncthreads();
      scan_bins(s, lane, wave);
    }
  }

  // the draw: weights by index
  if (last > -INFINITY || min_p > 0.f) {
    // a logit below this is too light (to a margin: its weight decides)
    const float cut = fmaxf(last, min_p > 0.f ? (float)((double)top + (double)temperature * (log((double)min_p) - 1e-6) -
                                                        1e-6 * fabs((double)top)) : -INFINITY);
    __syncthreads();
    if (threadIdx.x == 0) s.count = 0;
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
    __syncthreads();
    row.each(lane, [&](float l, int index) {
      if (l >= cut && inside(l, index)) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kList) s.list[at] = place_of(key_of(l), index);
      }
    });
    __syncthreads();
    const int n = s.count;
    if (n <= kList) {
      int shift = 0;
      while ((a.vocab - 1) >> shift >= kBins) ++shift;
      const auto light = [&](uint64_t place) {
        const uint64_t w = weight(of_key((uint32_t)(place >> 32)));
        return too_light(w) ? 0 : w;
      };
      for (int i = threadIdx.x; i < n; i += TH) add_to(s.bins[~(uint32_t)s.list[i] >> shift], light(s.list[i]));
      __syncthreads();
      const uint64_t total = scan_bins(s, lane, wave), target = target_of(total);
      for (int i = threadIdx.x; i < kBins; i += TH)
        if (target < s.bins[i] && target >= (i ? s.bins[i - 1] : 0)) s.at = i;
      uint64_t held[kList / TH];
#pragma unroll
      for (int e = 0; e < kList / TH; ++e) held[e] = (int)threadIdx.x + e * TH < n ? s.list[threadIdx.x + e * TH] : 0;
      if (threadIdx.x == 0) s.count = 0;
      __syncthreads();
      const int at = s.at;
      const uint64_t begin = at ? s.bins[at - 1] : 0;
#pragma unroll
      for (int e = 0; e < kList / TH; ++e)
        if ((int)threadIdx.x + e * TH < n && (int)(~(uint32_t)held[e] >> shift) == at && light(held[e]))
          s.list[atomicAdd(&s.count, 1)] = held[e];
      __syncthreads();
      const int m = s.count;
      if (m <= kSorted) {
        draw_list(m, begin, total);
        return;
      }
    }
  }
  const auto drawn = [&](float l, int index) -> uint64_t {
    if (!inside(l, index)) return 0;
    const uint64_t w = weight(l);
    return too_light(w) ? 0 : w;
  };
  // sums of the weights of 64 vectors each, or of a power of two of them
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
  __syncthreads();
  const int sets = (row.all + 63) / 64;
  int shift = 0;
  while ((sets - 1) >> shift >= kBins) ++shift;
  const auto set_sum = [&](int set, uint64_t(&w)[Row<T, WAVES>::V], typename Row<T, WAVES>::VT& v) {
    uint64_t sum = 0;
    const int vec = set * 64 + lane;
    if (vec < row.all) {
      v = row.load(vec);
#pragma unroll
      for (int j = 0; j < Row<T, WAVES>::V; ++j) sum += w[j] = drawn(fmaxf((float)v[j], -INFINITY), row.first(vec) + j);
    }
    return sum;
  };
#pragma unroll 2
  for (int set = wave; set < sets; set += WAVES) {
    uint64_t w[Row<T, WAVES>::V];
    typename Row<T, WAVES>::VT v;
    const uint64_t sum = wave_sum(set_sum(set, w, v));
    if (lane == 0) add_to(s.bins[set >> shift], sum);
  }
  __syncthreads();
  const uint64_t total = scan_bins(s, lane, wave), target = target_of(total);
  for (int i = threadIdx.x; i < kBins; i += TH)
    if (target < s.bins[i] && target >= (i ? s.bins[i - 1] : 0)) s.at = i;
  __syncthreads();
  if (wave) return;
  const int at = s.at;
  uint64_t begin = at ? s.bins[at - 1] : 0;
  for (int set = at << shift; set < min(sets, (at + 1) << shift); ++set) {
    uint64_t w[Row<T, WAVES>::V];
    typename Row<T, WAVES>::VT v;
    const uint64_t sum = set_sum(set, w, v), upto = wave_scan(sum, lane), all = lane64(upto, 63);
    if (target < begin + all) {
      uint64_t from = begin + upto - sum;
      if (target >= from && target < from + sum) {
#pragma unroll
        for (int j = 0; j < Row<T, WAVES>::V; ++j) {
          if (target >= from && target < from + w[j]) finish(row.first(set * 64 + lane) + j, fmaxf((float)v[j], -INFINITY), total);
          from += w[j];
        }
      }
      return;
    }
    begin += all;
  }
}

template <class T>
int sample_run(const SampleArgs& a, int rows, hipStream_t s) {
  if (a.vocab <= 8192)
    NHIP_LAUNCH("sample", (sample_kernel<T, 4>), dim3((uint32_t)rows), dim3(256), 0, s, a);
  else
    NHIP_LAUNCH("sample", (sample_kernel<T, 16>), dim3((uint32_t)rows), dim3(1024), 0, s, a);
  return check_launch("sample");
}

int sample_args(const nhip_sample_desc* d) {
  if (!d) return fail(NHIP_STATUS_NULL_POINTER, "sample: null descriptor");
  if (!elem_size(d->dtype)) return fail(NHIP_STATUS_UNSUPPORTED, "sample: dtype has to be F32, F16 or BF16");
  if (d->rows < 0 || d->vocab <= 0) return fail(NHIP_STATUS_INVALID_SHAPE, "sample: a row holds at least one logit");
  if (d->vocab > 1 << 30) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "sample: at most 2^30 logits to a row");
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
  *bytes = 0;
  return ok();
}

int nhip_sample_forward(const nhip_sample_desc* desc, const void* logits, const float* uniform, int32_t* token,
                        float* logprob, void* workspace, uint64_t workspace_bytes, void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  NHIP_TRY(sample_args(desc));
  if (desc->rows == 0) return ok();
  if (!logits || !uniform || !token || !logprob) return fail(NHIP_STATUS_NULL_POINTER, "sample: null pointer");
  if (!aligned_to(logits, elem_size(desc->dtype)) || !aligned_to(uniform, 4) || !aligned_to(token, 4) || !aligned_to(logprob, 4))
    return fail(NHIP_STATUS_CONSTRAINT_VIOLATION, "sample: a tensor is not aligned to its type");
  const SampleArgs a{logits,           desc->row_stride,       desc->vocab,      uniform,          desc->temperature,
                     desc->top_p,      desc->min_p,            desc->top_k,      desc->temperature_each,
                     desc->top_k_each, desc->top_p_each,       desc->min_p_each, token,            logprob};
  return NHIP_FOR_ELEM(desc->dtype, T, sample_run<T>(a, desc->rows, as_stream(stream)));
}

}  // extern "C"
