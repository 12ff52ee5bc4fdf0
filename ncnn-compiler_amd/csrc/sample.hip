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

constexpr int kBins = 1024;   // of weights' exponents, width kRange / kBins
constexpr int kList = 4096;   // tokens that LDS holds in order
constexpr int kMaxListK = 1024;
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

// exp((l - top) / T) in units of 2^-44, to the nearest: 2^t as 2^n times the
// Taylor series of e^(f ln 2) for |f| <= 1/2, whose first term left out is 6e-15.
struct Weights {
  double top, rate;  // log2(e) / T
  __device__ __forceinline__ uint64_t operator()(float l) const {
    const double x = (double)l - top;
    if (x >= 0 || l == (float)top) return uint64_t(1) << 44;  // (infinity less infinity)
    const double t = x * rate;
    if (!(t > -46.0)) return 0;
    const double n = __builtin_rint(t), f = t - n;
    constexpr double kLn2 = 0.69314718055994530942;
    const double z = f * kLn2;
    double p = 1.0 / 39916800;
    p = fma(p, z, 1.0 / 3628800);
    p = fma(p, z, 1.0 / 362880);
    p = fma(p, z, 1.0 / 40320);
    p = fma(p, z, 1.0 / 5040);
    p = fma(p, z, 1.0 / 720);
    p = fma(p, z, 1.0 / 120);
    p = fma(p, z, 1.0 / 24);
    p = fma(p, z, 1.0 / 6);
    p = fma(p, z, 0.5);
    p = fma(p, z, 1.0);
    p = fma(p, z, 1.0);
    // p 2^(n + 44) + 2^52: the sum's last 52 bits are the whole number
    const double scale = __builtin_bit_cast(double, (uint64_t)(1023 + 44 + (int)n) << 52);
    return __builtin_bit_cast(uint64_t, fma(p, scale, 4503599627370496.0)) & ((uint64_t(1) << 52) - 1);
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

// A row in 16-byte vectors from the aligned place at or before its start, dealt
// to the waves in runs; what lies outside the row is -infinity and is not read.
// NaN is -infinity.
template <class T, int WAVES>
struct Row {
  static constexpr int V = kVec<T>;
  typedef T VT __attribute__((ext_vector_type(V)));
  const T* from;  // aligned
  int shift, vocab, begin, end;  // the wave's vectors
  __device__ __forceinline__ Row(const T* row, int vocab, int wave) : vocab(vocab) {
    shift = (int)(((uintptr_t)row & 15) / sizeof(T));
    from = row - shift;
    const int all = (int)(((int64_t)vocab + shift + V - 1) / V), each = (all + WAVES * 64 - 1) / (WAVES * 64) * 64;
    begin = min(wave * each, all);
    end = min(begin + each, all);
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
  uint64_t part[WAVES];
  uint32_t keys[WAVES];
  int32_t count, at;
  uint64_t before;
};

// list[0 .. count) in falling order; count at most kList.
template <int TH>
__device__ __forceinline__ void sort_list(uint64_t* list, int count) {
  int size = 2;
  while (size < count) size <<= 1;
  for (int i = count + threadIdx.x; i < size; i += TH) list[i] = 0;
  __syncthreads();
  for (int run = 2; run <= size; run <<= 1)
    for (int gap = run >> 1; gap; gap >>= 1) {
      for (int i = threadIdx.x; i < size / 2; i += TH) {
        const int a = (i / gap) * gap * 2 + i % gap, b = a + gap;
        const uint64_t x = list[a], y = list[b];
        if ((x < y) == ((a & run) == 0)) {
          list[a] = y;
          list[b] = x;
        }
      }
      __syncthreads();
    }
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
// ones, leaves a few hundred, which are sorted in LDS.  Otherwise a histogram of
// the tokens by their weights' exponents, of counts for top-k and of masses for
// top-p, says in which bin the border lies; its tokens are sorted in LDS, or if
// they are too many (equal logits) the bin is divided further by the logits' bits.
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
  // a bound that at least `want` tokens of each wave reach: its lanes' want-th largest
  uint32_t bound = 0;
  if (k <= kMaxListK && k < a.vocab) {
    const int want = (k + WAVES - 1) / WAVES;
    const uint32_t key = key_of(mine);
    for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
      if (__popcll(__ballot(key >= (bound | bit))) >= want) bound |= bit;
  }
  if (lane == 0) {
    s.part[wave] = key_of(top);
    s.keys[wave] = bound;
  }
  if (threadIdx.x == 0) s.count = 0;
  for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
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
  const Weights weight{(double)top, 1.4426950408889634074 / (double)(temperature > 0.f ? temperature : 1.f)};
  const float reach = kRange * temperature;  // tokens further below the largest weigh nothing
  const double u = fmin(fmax((double)a.uniform[r], 0.0), 1.0 - 0x1p-53);  // NaN: 0
  const auto finish = [&](int index, float l, uint64_t total) {
    const double x = l == top ? 0.0 : ((double)l - (double)top) / (double)temperature;
    a.token[r] = index;
    a.logprob[r] = (float)(x - log((double)total * 0x1p-44));
  };
  // the first whose cumulated weight is past this
  const auto target_of = [&](uint64_t total) { return min((uint64_t)((double)total * u), total - 1); };

  if (k <= kMaxListK && k < a.vocab) {
    // ------------------------------------------------ few tokens are kept
    const float least = k == 1 ? top : fmaxf(of_key(bound), top - reach);
    row.each(lane, [&](float l, int index) {
      if (l >= least && l != -INFINITY) {
        const int at = atomicAdd(&s.count, 1);
        if (at < kList) s.list[at] = place_of(key_of(l), index);
      }
    });
    __syncthreads();
    int count = s.count;
    if (k == 1 && count > kList) {
      // equal ones past the list: the lowest index of each lane
      __syncthreads();
      int low = 0x7fffffff;
      row.each(lane, [&](float l, int index) {
        if (l == top) low = min(low, index);
      });
      s.list[threadIdx.x] = place_of(top_key, low);
      count = TH;
      __syncthreads();
    }
    if (count <= kList) {
      if (k == 1) {
        uint64_t best = 0;
        for (int i = threadIdx.x; i < count; i += TH) best = max(best, s.list[i]);
#pragma unroll
        for (int o = 32; o; o >>= 1) best = max(best, shfl_xor64(best, o));
        if (lane == 0) s.part[wave] = best;
        __syncthreads();
        if (threadIdx.x == 0) {
#pragma unroll
          for (int w = 1; w < WAVES; ++w) best = max(best, s.part[w]);
          finish((int)~(uint32_t)best, top, uint64_t(1) << 44);
        }
        return;
      }
      sort_list<TH>(s.list, count);
      const int n = min(k, count);
      // top-p and min-p: the bins hold the weights' sums up to each
      for (int i = threadIdx.x; i < n; i += TH) s.bins[i] = weight(of_key((uint32_t)(s.list[i] >> 32)));
      __syncthreads();
      uint64_t total = scan_bins(s, lane, wave);
      const double limit = top_p < 1.f ? (double)top_p * (double)total : INFINITY;
      if (threadIdx.x == 0) s.at = 1;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += TH) {
        const uint64_t before = i ? s.bins[i - 1] : 0, w = s.bins[i] - before;
        const bool stays = (double)before < limit && (double)w * 0x1p-44 >= (double)min_p;
        if (stays && w) atomicMax(&s.at, i + 1);
      }
      __syncthreads();
      const int kept = s.at;
      total = s.bins[kept - 1];
      __syncthreads();
      // in the order of the indices
      for (int i = threadIdx.x; i < kept; i += TH) {
        const uint64_t p = s.list[i];
        s.list[i] = p << 32 | p >> 32;  // the index turned round, so falling order is rising index
      }
      __syncthreads();
      sort_list<TH>(s.list, kept);
      for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = i < kept ? weight(of_key((uint32_t)s.list[i])) : 0;
      __syncthreads();
      scan_bins(s, lane, wave);
      const uint64_t target = target_of(total);
      for (int i = threadIdx.x; i < kept; i += TH) {
        const uint64_t upto = s.bins[i];
        if (upto > target && (i ? s.bins[i - 1] : 0) <= target)
          finish((int)~(uint32_t)(s.list[i] >> 32), of_key((uint32_t)s.list[i]), total);
      }
      return;
    }
  }

  // --------------------------------------------------- any number is kept
  // everything up to `last` of the order, as far as it weighs anything
  uint64_t last = 0;
  const float rate = (float)kBins / reach;
  const auto bin_of = [&](float l) { return l == top ? 0 : (int)fminf((top - l) * rate, (float)(kBins - 1)); };
  const auto inside = [&](float l, int index) {
    return (l == top || top - l <= reach) && l != -INFINITY && place_of(key_of(l), index) >= last;
  };
#pragma unroll 1
  for (int by = 0; by < 2; ++by) {  // top-k by count, then top-p by weight
    if (by == 0 ? k == a.vocab : !(top_p < 1.f)) continue;
    const auto measure = [&](float l) { return by ? weight(l) : (uint64_t)1; };
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
    __syncthreads();
    row.each(lane, [&](float l, int index) {
      if (inside(l, index))
        if (const uint64_t m = measure(l)) atomicAdd((unsigned long long*)&s.bins[bin_of(l)], (unsigned long long)m);
    });
    __syncthreads();
    const uint64_t all = scan_bins(s, lane, wave);
    const double limit = by ? fmax((double)top_p * (double)all, 1.0) : (double)k;  // (the first one always)
    // kept: those with less than `limit` before them; the last of them lies in the bin that reaches it
    if ((double)all < limit || (by == 0 && all <= (uint64_t)k)) continue;
    uint64_t before = 0;          // the measure of what comes before the present bin
    uint32_t low = 0, high = 0;   // its keys
    bool keys = false;            // by keys, not yet: the bin of weights `bin`
    int bin = 0, shift = 0;
    for (;;) {
      // the first bin with which the sum reaches the limit (or the first that holds anything)
      if (threadIdx.x == 0) s.at = kBins - 1;
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += TH)
        if ((double)(before + s.bins[i]) >= limit && s.bins[i]) atomicMin(&s.at, i);
      if (threadIdx.x == 0) s.count = 0;
      __syncthreads();
      const int at = s.at;
      if (!keys) {
        bin = at;
      } else {
        // bins of keys: the largest first
        const uint64_t width = uint64_t(1) << shift;
        const uint32_t h = high;
        high = h - (uint32_t)(at * width);
        low = (uint64_t)(high - low) >= width ? (uint32_t)(high - (width - 1)) : low;
      }
      before += at ? s.bins[at - 1] : 0;
      __syncthreads();
      const auto here = [&](float l, int index) {
        if (!inside(l, index)) return false;
        const uint32_t key = key_of(l);
        return bin_of(l) == bin && (!keys || (key >= low && key <= high));
      };
      uint32_t most = 0, least = 0xffffffffu;
      row.each(lane, [&](float l, int index) {
        if (here(l, index) && (!by || measure(l))) {
          const uint32_t key = key_of(l);
          most = max(most, key);
          least = min(least, key);
          const int i = atomicAdd(&s.count, 1);
          if (i < kList) s.list[i] = place_of(key, index);
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
      if (count <= kList) {
        sort_list<TH>(s.list, count);
        // by kBins at a time: the last with less than the limit before it
        for (int i0 = 0; i0 < count; i0 += kBins) {
          for (int i = threadIdx.x; i < kBins; i += TH)
            s.bins[i] = i0 + i < count ? measure(of_key((uint32_t)(s.list[i0 + i] >> 32))) : 0;
          if (threadIdx.x == 0) s.at = -1;
          __syncthreads();
          const uint64_t sum = scan_bins(s, lane, wave);
          for (int i = threadIdx.x; i < min(kBins, count - i0); i += TH)
            if ((double)(before + (i ? s.bins[i - 1] : 0)) < limit) atomicMax(&s.at, i);
          __syncthreads();
          const int i = s.at;
          if (i >= 0) last = s.list[i0 + i];
          before += sum;
          __syncthreads();
          if (i < min(kBins, count - i0) - 1) break;
        }
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
        const uint64_t m = measure(of_key(low));
        const double over = (limit - (double)before) / (double)m;
        const int keep = (int)fmax(1.0, fmin(ceil(over), (double)count));
        int held = 0;
        row.each(lane, [&](float l, int index) { held += here(l, index) && key_of(l) == low; });
        const uint64_t wave_held = wave_sum((uint64_t)held);
        if (lane == 0) s.part[wave] = wave_held;
        if (threadIdx.x == 0) s.before = 0;
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
              for (int j = 0; j < Row<T, WAVES>::V; ++j) {
                const float l = fmaxf((float)v[j], -INFINITY);
                n += here(l, row.first(c + lane) + j) && key_of(l) == low;
              }
            }
            const int upto = (int)wave_scan((uint64_t)n, lane);
            if (upto >= left && upto - n < left) {
              int need = left - (upto - n);
#pragma unroll
              for (int j = 0; j < Row<T, WAVES>::V; ++j) {
                const float l = fmaxf((float)v[j], -INFINITY);
                if (here(l, row.first(c + lane) + j) && key_of(l) == low && --need == 0)
                  s.before = place_of(low, row.first(c + lane) + j);
              }
            }
            const int all_here = __builtin_amdgcn_readlane(upto, 63);
            if (all_here >= left) break;
            left -= all_here;
          }
        }
        __syncthreads();
        last = s.before;
        break;
      }
      // the bin's keys, largest first, into kBins parts
      keys = true;
      shift = 0;
      while (((uint64_t)(high - low) >> shift) >= kBins) ++shift;
      for (int i = threadIdx.x; i < kBins; i += TH) s.bins[i] = 0;
      __syncthreads();
      const uint32_t h = high, lo = low;
      row.each(lane, [&](float l, int index) {
        if (!inside(l, index) || bin_of(l) != bin) return;
        const uint32_t key = key_of(l);
        if (key < lo || key > h) return;
        if (const uint64_t m = measure(l)) atomicAdd((unsigned long long*)&s.bins[(h - key) >> shift], (unsigned long long)m);
      });
      __syncthreads();
      scan_bins(s, lane, wave);
    }
  }

  // the draw: weights by index
  const auto drawn = [&](float l, int index) -> uint64_t {
    if (!inside(l, index)) return 0;
    const uint64_t w = weight(l);
    return (double)w * 0x1p-44 < (double)min_p ? 0 : w;
  };
  uint64_t mass = 0;
  row.each(lane, [&](float l, int index) { mass += drawn(l, index); });
  mass = wave_sum(mass);
  __syncthreads();
  if (lane == 0) s.part[wave] = mass;
  __syncthreads();
  uint64_t total = 0, begin = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) begin += s.part[w];
    total += s.part[w];
  }
  const uint64_t target = target_of(total);
  if (target < begin || target >= begin + mass) return;
  for (int c = row.begin; c < row.end; c += 64) {
    uint64_t w[Row<T, WAVES>::V], sum = 0;
    typename Row<T, WAVES>::VT v;
    if (c + lane < row.end) {
      v = row.load(c + lane);
#pragma unroll
      for (int j = 0; j < Row<T, WAVES>::V; ++j) sum += w[j] = drawn(fmaxf((float)v[j], -INFINITY), row.first(c + lane) + j);
    }
    const uint64_t upto = wave_scan(sum, lane), all = lane64(upto, 63);
    if (target < begin + all) {
      uint64_t at = begin + upto - sum;
      if (target >= at && target < at + sum) {
#pragma unroll
        for (int j = 0; j < Row<T, WAVES>::V; ++j) {
          if (target >= at && target < at + w[j]) finish(row.first(c + lane) + j, fmaxf((float)v[j], -INFINITY), total);
          at += w[j];
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
