// Attention kernels, instantiated once for each element type
// (attn_f32.hip, attn_f16.hip, attn_bf16.hip).
//
// A key/value head's query rows (queries x the heads that share it, row =
// query * group + head) are one matrix, so that grouped heads read keys and
// values once.  Scores are formed transposed, S^T = K Q^T: a lane then holds
// scores of one row (its column), the softmax's statistics are one number a
// lane, and the probabilities already lie as the second product
// O^T = V^T P^T takes its right operand.
#pragma once

#include <type_traits>

#include "elem.h"
#include "kv_cache8.h"

namespace nhip {

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t qs[3], ks[3], vs[3];  // batch, token, head
  Kv8 cache;
  const int32_t* lengths;
  const uint8_t* mask;
  int64_t mask_stride;
  int32_t batch, queries, keys, heads, kv_heads, group, d, causal;
  int32_t rows;       // queries * group
  int32_t tiles;      // the kernel of many rows
  int32_t row_tiles;  // row tiles of a key/value head
  int32_t reps;       // few rows: times 16 rows of a workgroup (2 only of own keys behind a prefix)
  int32_t splits;     // few rows: parts of a sequence's keys
  int32_t workers;    // many rows: workgroups
  int32_t units;      // and the parts of a row tile's keys that are dealt to them
  int32_t parts;      // the results stay parts, also where there is one to a row
  int32_t per;        // queries come in runs of `per`, q_run elements apart (0: one run)
  int64_t q_run;
  float scale_log2;   // scale / ln 2
  float* part_o;      // few rows: [batch][kv_heads][rows][splits][d]; many: [workers][2][128][d] ([workers + row tiles][128][d] if all are parts)
  float2* part_ml;    // the same without [d]: maximum, sum
};

// Where keys and values come from.
enum { kSrcVec = 0, kSrcAny = 1, kSrcInt8 = 2 };  // 16-byte aligned rows; any strides; the 8-bit cache

int attn_run_f32(const AttnArgs& a, int src, hipStream_t s);
int attn_run_f16(const AttnArgs& a, int src, hipStream_t s);
int attn_run_bf16(const AttnArgs& a, int src, hipStream_t s);
// Over the 8-bit cache: the parts of `prefix`, whose sequences are groups of
// those of `own` in turn (their queries one behind the other), and of `own`,
// joined to the results of `own`.
int attn_prefix_f32(const AttnArgs& prefix, const AttnArgs& own, hipStream_t s);
int attn_prefix_f16(const AttnArgs& prefix, const AttnArgs& own, hipStream_t s);
int attn_prefix_bf16(const AttnArgs& prefix, const AttnArgs& own, hipStream_t s);

namespace attn {

constexpr int kRowTile = 16;   // query rows of a workgroup
constexpr int kKeyTile = 32;   // keys of a wave's step
constexpr int kWaves = 4;
constexpr int kTilesRows = 32 * kWaves;  // query rows of a workgroup, many rows

typedef short v4s __attribute__((ext_vector_type(4)));

template <class T>
struct Frag;  // eight values of an operand
template <>
struct Frag<float> {
  typedef v8f type;
};
template <>
struct Frag<f16> {
  typedef v8h type;
};
template <>
struct Frag<bf16> {
  typedef v8b type;
};

// 16 x 16 += A [16 x 32] B [32 x 16].  Lane l holds eight values of row
// (column) l & 15, and of the sum column l & 15, rows 4 (l >> 4) .. + 3.  Any
// assignment of the summed index to (lane group, place) serves, as long as A
// and B have the same: fp32 takes the eight places one at a time.
__device__ __forceinline__ v4f mma16(v8b a, v8b b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mma16(v8h a, v8h b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mma16(v8f a, v8f b, v4f c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// 32 x 32 += A [32 x 16] B [16 x 32].  Lane l holds eight values of row (column)
// l & 31, and of the sum column l & 31, rows 8 (i / 4) + 4 (l >> 5) + i % 4.
__device__ __forceinline__ v16f mma32(v8b a, v8b b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f mma32(v8h a, v8h b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v16f mma32(v8f a, v8f b, v16f c) {
#pragma unroll
  for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// A matrix instruction's sums may be read some 20 cycles after it at the
// earliest, and no hardware waits for them.  The compiler counts the cycles
// along straight code; where a branch may follow (one around a load, say), its
// count was seen to miss the path on which the branch is taken.  So sums pass
// through this before any branch.
template <class V>
__device__ __forceinline__ void settle(V& sums) {
  asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sums));
}
template <class V>
__device__ __forceinline__ void settle(V& sums, V& more) {
  asm volatile("s_nop 15\n\ts_nop 7" : "+v"(sums), "+v"(more));
}
// Query qi's place among a sequence's queries.
__device__ __forceinline__ int64_t query_at(const AttnArgs& a, int qi) {
  return a.per ? qi / a.per * a.q_run + qi % a.per * a.qs[1] : qi * a.qs[1];
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

template <class T>
__device__ __forceinline__ typename Frag<T>::type zero_frag() {
  typename Frag<T>::type f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (T)0.f;
  return f;
}

// Eight channels from c of a query row; channels at and past d are 0.  VEC:
// the row is 16-byte aligned and d a multiple of 8 (4 for fp32).
template <class T, bool VEC>
__device__ __forceinline__ typename Frag<T>::type load_q(const T* row, int c, int d) {
  typename Frag<T>::type f = zero_frag<T>();
  if constexpr (VEC && sizeof(T) == 2) {
    if (c < d) f = *reinterpret_cast<const typename Frag<T>::type*>(row + c);
  } else if constexpr (VEC) {
#pragma unroll
    for (int j = 0; j < 8; j += 4)
      if (c + j < d) {
        const v4f v = *reinterpret_cast<const v4f*>(row + c + j);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[j + i] = v[i];
      }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < d) f[i] = row[c + i];
  }
  return f;
}

// Sixteen codes as T (exact in every type): the first or last eight.
template <class T>
__device__ __forceinline__ typename Frag<T>::type codes8(uint32_t lo, uint32_t hi) {
  typename Frag<T>::type f;
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = (T)(float)(int8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
  return f;
}

// Few rows: type of probabilities and values in the second product, and the
// parts that a probability is the sum of.  16-bit types take one, a rounding
// (the error against 64 bits is 2.3e-3 of the result's norm in bf16, where rounding
// the result alone leaves 1.7e-3; 2.9e-4 and 2.1e-4 in fp16).  A second part takes up to
// 3% more time, over the cache 1 to 6% (64 samples behind four prefixes of 3136 keys 37.7 ->
// 38.5 us), but it may be 0 or negative, and an
// infinite value that it meets NaN.  The sum l is of the probabilities as they
// were.  Codes times probabilities times a page's scale may leave fp16's range,
// so fp16 queries over the cache take bf16, which needs both parts for fp16's
// digits, and codes are finite.
template <class T, int SRC>
struct Second {
  typedef T type;
  static constexpr int parts = 1;
};
template <>
struct Second<f16, kSrcInt8> {
  typedef bf16 type;
  static constexpr int parts = 2;
};

// Row r of a tile that starts at key0 (uniform), channels from c: one 16-byte
// load without a branch.  A row that does not count, or c at or past d, is
// sent out of the buffer's range and reads as 0, whatever memory holds there.
// `page` (cache only, uniform): the row's page.
template <class T, int SRC>
__device__ __forceinline__ int4 load_row16(const AttnArgs& a, const void* base, int64_t stride, const int8_t* codes,
                                           int kvh, int64_t page, int key0, int r, int c, bool counts) {
  if constexpr (SRC == kSrcInt8) {
    // a chunk may run past channel d into the next row, or past the page's end, where the buffer ends
    const uint32_t bytes = (uint32_t)a.d << a.cache.shift;
    const int8_t* at = codes + (page < 0 ? 0 : page * a.cache.kv_heads + kvh) * bytes;
    const uint32_t slot = (key0 + r) & ((1 << a.cache.shift) - 1), off = slot * a.d + c;
    return buf_load_b128(make_rsrc(at, bytes), counts && c < a.d ? off : kBufOOB);
  } else {
    const T* at = (const T*)base + (int64_t)key0 * stride;
    const uint32_t off = (r * (uint32_t)stride + c) * (uint32_t)sizeof(T);
    return buf_load_b128(make_rsrc(at, 0x7fffffffu), counts && c < a.d ? off : kBufOOB);
  }
}

// The same eight channels of rows of any stride and alignment, an element at a time: always from a place inside the tensor.
template <class T>
__device__ __forceinline__ typename Frag<T>::type load_any8(const AttnArgs& a, const T* base, int64_t stride, int key,
                                                            int first, int c, bool counts) {
  const T* row = base + (int64_t)(counts ? key : first) * stride;
  typename Frag<T>::type f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const T v = row[min(c + i, a.d - 1)];
    f[i] = counts && c + i < a.d ? v : (T)0.f;
  }
  return f;
}

// A tile's keys as the lanes know them, a key to a lane (from 0; lanes past the tile repeat it).
struct TileKeys {
  uint64_t counts;       // bit i: key i counts
  int64_t page;          // cache: the lane's key's page, its scales
  float kscale, vscale;
};

// First half of learning about a tile: loads only.
struct TileAsk {
  int32_t id;
  uint8_t on;
};
template <int SRC, int KEYS>
__device__ __forceinline__ TileAsk ask_tile(const AttnArgs& a, int b, int key0, int lane) {
  TileAsk t{0, 1};
  const int key = min(key0 + (lane & (KEYS - 1)), a.keys - 1);
  if constexpr (SRC == kSrcInt8) {
    const int64_t page = key >> a.cache.shift;
    const bool in = page < a.cache.table_pages;
    t.id = a.cache.table_pages ? a.cache.table[b * a.cache.table_pages + (in ? page : 0)] : -1;
    if (!in) t.id = -1;
  } else if (a.mask) {
    t.on = a.mask[b * a.mask_stride + key];
  }
  return t;
}
template <int SRC, int KEYS>
__device__ __forceinline__ TileKeys know_tile(const AttnArgs& a, TileAsk t, int kvh, int key0, int end, int lane) {
  TileKeys k{0, 0, 1.f, 1.f};
  bool counts = key0 + (lane & (KEYS - 1)) < end && t.on;
  if constexpr (SRC == kSrcInt8) {
    const bool there = t.id >= 0 && t.id < a.cache.pages;
    counts = counts && there;
    k.page = there ? t.id : -1;
    if (a.cache.pages) {
      const int64_t at = (there ? (int64_t)t.id : 0) * a.cache.kv_heads + kvh;
      k.kscale = a.cache.k_scale[at];
      k.vscale = a.cache.v_scale[at];
    }
    // (Products take the scale of a page's first key.  A page of which no row
    // sees a token may hold any scale; one that is not finite, times a probability
    // of 0, would be NaN.)
    if (!there || key0 + (lane & (KEYS - 1)) >= end) k.kscale = k.vscale = 0.f;
  }
  k.counts = __ballot(counts);
  return k;
}
__device__ __forceinline__ int64_t lane_page(const TileKeys& k, int lane) {
  return __builtin_amdgcn_readlane((int)k.page, lane);  // page numbers are int32
}
__device__ __forceinline__ float lane_float(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// The largest / the sum of a value over the lanes that hold the same row's
// other keys: lanes l ^ 32, and of 16 x 16 tiles l ^ 16 too.
// (The swaps stand in assembly: from the builtin, both results of equal operands
// were taken for equal, and the maximum for either.  They need two cycles
// after the write of an operand.)
__device__ __forceinline__ float max32(float v) {
  float w = v;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(v), "+v"(w));
  return fmaxf(v, w);
}
__device__ __forceinline__ float max16(float v) {
  float w = v;
  asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
  return fmaxf(v, w);
}

// Keys [begin, end) of one part of a sequence, of which a workgroup's last
// row sees `visible`; parts are whole multiples of `unit`.
__device__ __forceinline__ void part_of(const AttnArgs& a, int length, int visible, int split, int unit, int& begin, int& end) {
  const int part = ((length + a.splits - 1) / a.splits + unit - 1) / unit * unit;
  begin = min(split * part, visible);
  end = min(begin + part, visible);
}

// ---------------------------------------------------------------- few rows
// A lane's eight summed values down one channel of V in LDS: places 0..3 from
// keys 4g .. 4g + 3, places 4..7 from keys 16 + 4g .. (g = lane / 16), the
// order in which two score tiles hold a row's keys.
template <class T, int STRIDE>
__device__ __forceinline__ typename Frag<T>::type load_v16(const T* tile, int c0, int lane) {
  const int g = lane >> 4, j = lane & 15;
  typename Frag<T>::type f;
  if constexpr (sizeof(T) == 2) {
    // transposing read: 16 lanes address 4 keys x 16 channels, 8 bytes each,
    // and lane j gets channel j of the four keys
    const T* at = tile + (4 * g + (j >> 2)) * STRIDE + c0 + (j & 3) * 4;
    typedef __attribute__((address_space(3))) v4s lds4;
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + 16 * STRIDE));
    f = __builtin_bit_cast(typename Frag<T>::type, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = tile[(16 * (i >> 2) + 4 * g + (i & 3)) * STRIDE + c0 + j];
  }
  return f;
}

// The exponent's reference point need not be the row's largest score: it moves
// only where a score lies more than kRoom above it, which spares most tiles the
// scaling of the sums, and then to kBelow under that score.  fp16
// probabilities lie high in their range (2^6 to 2^14 for the largest), so that
// small ones keep their digits: they decide where the large ones meet values of 0.
template <class P>
constexpr float kRoom = std::is_same<P, f16>::value ? 14.f : 8.f;
template <class P>
constexpr float kBelow = std::is_same<P, f16>::value ? 6.f : 0.f;

template <class P>
constexpr int kPad16 = sizeof(P) == 2 ? 16 : 4;  // the rows that a read takes together lie in different banks

// Workgroups that a CU is to hold, what the registers are dealt out for: few
// rows over the cache wait for memory and convert codes in turn (a cached step
// 79 us with two, 73 with three).
constexpr int rows_per_cu(int size, int dp, int src) {
  return src == kSrcInt8 ? (size == 2 && dp <= 128 ? 3 : 1) : (src == kSrcVec && size * dp <= 256 ? 2 : 1);
}

template <class T, int DP, int SRC>
constexpr int rows_lds() {
  typedef typename Second<T, SRC>::type P;
  constexpr int tile = kWaves * kKeyTile * (DP + kPad16<P>) * (int)sizeof(P);
  constexpr int merge = kWaves * kRowTile * (DP + 4 + 4) * 4;
  return tile > merge ? tile : merge;
}

// One wave's next 32 keys and values on their way.
template <class T, int DP, int SRC>
struct RowsTile {
  typedef typename Second<T, SRC>::type P;
  static constexpr int E = SRC == kSrcInt8 ? 16 : 16 / (int)sizeof(T);  // channels of a 16-byte load
  static constexpr int KL = DP / (4 * E);        // loads of a key row's channels for one lane group
  static constexpr int VL = kKeyTile * DP / E / 64;
  TileKeys keys;
  // kSrcAny holds whole fragments, the others 16-byte pieces
  int4 k[2][SRC == kSrcAny ? 1 : KL], v[SRC == kSrcAny ? 1 : VL];
  typename Frag<T>::type ka[2][SRC == kSrcAny ? DP / 32 : 1], va[SRC == kSrcAny ? kKeyTile * DP / 8 / 64 : 1];

  // Channel from which lane group g's piece p of a key row starts: pieces of
  // 16 bytes; fp32 takes two to a fragment, codes two fragments to a piece.
  __device__ __forceinline__ static int k_channel(int p, int g) {
    if constexpr (SRC == kSrcInt8) return p * 64 + g * 16;
    if constexpr (sizeof(T) == 4) return (p >> 1) * 32 + g * 8 + (p & 1) * 4;
    return p * 32 + g * 8;
  }
  // ... and the one from which fragment s does.
  __device__ __forceinline__ static int q_channel(int s, int g) {
    return SRC == kSrcInt8 ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
  }

  __device__ __forceinline__ void load(const AttnArgs& a, const T* kbase, const T* vbase, int kvh, int key0, int first, int lane) {
    const int g = lane >> 4, col = lane & 15;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bool on = keys.counts >> (t * 16 + col) & 1;
      if constexpr (SRC == kSrcAny) {
#pragma unroll
        for (int s = 0; s < DP / 32; ++s) ka[t][s] = load_any8(a, kbase, a.ks[1], key0 + t * 16 + col, first, s * 32 + g * 8, on);
      } else {
        const int64_t page = SRC == kSrcInt8 ? lane_page(keys, t * 16) : 0;
#pragma unroll
        for (int p = 0; p < KL; ++p)
          k[t][p] = load_row16<T, SRC>(a, kbase, a.ks[1], a.cache.k, kvh, page, key0, t * 16 + col, k_channel(p, g), on);
      }
    }
    if constexpr (SRC == kSrcAny) {
#pragma unroll
      for (int i = 0; i < kKeyTile * DP / 8 / 64; ++i) {
        const int at = lane + 64 * i, r = at / (DP / 8);
        va[i] = load_any8(a, vbase, a.vs[1], key0 + r, first, at % (DP / 8) * 8, keys.counts >> r & 1);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        constexpr int per = DP / E;  // pieces of a row; the 64 of one load lie inside 16 rows
        const int at = lane + 64 * i, r = at / per;
        const int64_t page = SRC == kSrcInt8 ? lane_page(keys, 64 * i / per / 16 * 16) : 0;
        v[i] = load_row16<T, SRC>(a, vbase, a.vs[1], a.cache.v, kvh, page, key0, r, at % per * E, keys.counts >> r & 1);
      }
    }
  }
  __device__ __forceinline__ typename Frag<T>::type k_frag(int t, int s) const {
    if constexpr (SRC == kSrcAny) return ka[t][s];
    if constexpr (SRC == kSrcInt8) {
      const int4 q = k[t][s >> 1];
      return s & 1 ? codes8<T>(q.z, q.w) : codes8<T>(q.x, q.y);
    }
    if constexpr (SRC == kSrcVec && sizeof(T) == 4) {
      struct { int4 lo, hi; } both{k[t][2 * s], k[t][2 * s + 1]};
      return __builtin_bit_cast(typename Frag<T>::type, both);
    }
    if constexpr (SRC == kSrcVec && sizeof(T) == 2) return __builtin_bit_cast(typename Frag<T>::type, k[t][s]);
  }
  template <int STRIDE>
  __device__ __forceinline__ void store_v(P* tile, int lane) const {
    if constexpr (SRC == kSrcAny) {
#pragma unroll
      for (int i = 0; i < kKeyTile * DP / 8 / 64; ++i) {
        const int at = lane + 64 * i;
        *reinterpret_cast<typename Frag<T>::type*>(tile + at / (DP / 8) * STRIDE + at % (DP / 8) * 8) = va[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < VL; ++i) {
        const int at = lane + 64 * i;
        P* to = tile + at / (DP / E) * STRIDE + at % (DP / E) * E;
        if constexpr (SRC == kSrcInt8) {
          *reinterpret_cast<typename Frag<P>::type*>(to) = codes8<P>(v[i].x, v[i].y);
          *reinterpret_cast<typename Frag<P>::type*>(to + 8) = codes8<P>(v[i].z, v[i].w);
        } else {
          *reinterpret_cast<int4*>(to) = v[i];
        }
      }
    }
  }
};

// Row `in` of the waves' 16, row orow of the key/value head's.
template <class T, int OS>
__device__ __forceinline__ void join_waves(const AttnArgs& a, const float* mo, const float2* ml, int in, int orow, int b, int kvh,
                                           int split, int lane) {
  if (orow >= a.rows) return;
  float top = -INFINITY, total = 0.f, w[kWaves];
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) top = fmaxf(top, ml[i * kRowTile + in].x);
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const float2 t = ml[i * kRowTile + in];
    nan |= t.y < 0.f;
    w[i] = t.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(t.x - top);
    total += t.x == -INFINITY ? 0.f : w[i] * t.y;
  }
  const bool none = top == -INFINITY;
  const int oq = orow / a.group, oh = kvh * a.group + orow % a.group;
  const int64_t prow = (((int64_t)b * a.kv_heads + kvh) * a.rows + orow) * a.splits + split;
  for (int c = lane; c < a.d; c += 64) {
    float o = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i)
      if (w[i] != 0.f) o += w[i] * mo[(i * kRowTile + in) * OS + c];
    if (a.splits > 1 || a.parts)
      a.part_o[prow * a.d + c] = o;
    else
      ((T*)a.o)[(((int64_t)b * a.queries + oq) * a.heads + oh) * a.d + c] = (T)(none ? (nan ? NAN : 0.f) : o / total);
  }
  if ((a.splits > 1 || a.parts) && lane == 0) a.part_ml[prow] = make_float2(top, none ? (nan ? -1.f : 0.f) : total);
}

// One workgroup: 16 query rows of one key/value head over one part of the
// keys, its four waves every fourth tile of 32 keys, joined at the end.  Keys
// go from memory to the registers that the products read, values through the
// wave's own LDS, which turns them; the next tile's loads are under way while
// one is worked on.  Reading keys and values bounds it: 32 sequences of 3136
// keys, 8 heads of 128 bf16 67 us a call (326 MB, 4.9 TB/s, a large copy's rate
// 5.2); over the cache 16 of 12544 keys 71 us (316 MB, 4.4 TB/s, 5 us of it the
// launch that joins the parts).
// R: times 16 rows of a workgroup, which share what is read and converted of the keys.
template <class T, int DP, int SRC, int R = 1>
__device__ __forceinline__ void rows_body(const AttnArgs& a, uint32_t at, char* lds) {
  typedef typename Second<T, SRC>::type P;
  typedef typename Frag<T>::type FT;
  typedef typename Frag<P>::type FP;
  typedef RowsTile<T, DP, SRC> Tile;
  constexpr int KS = DP / 32, DT = DP / 16, STRIDE = DP + kPad16<P>, STEP = kWaves * kKeyTile, ROWS = kRowTile * R;
  const int lane = threadIdx.x & 63, wave = wave_id(), g = lane >> 4, col = lane & 15;
  const int rt = at % a.row_tiles;
  at /= a.row_tiles;
  const int split = at % a.splits;
  at /= a.splits;
  const int kvh = at % a.kv_heads, b = at / a.kv_heads;

  const int length = a.lengths ? max(0, min(a.lengths[b], a.keys)) : a.keys;
  // keys that the lane's rows see, and that any row of the tile does
  int sees[R], all_see = length, visible = length, begin, end;
  FT qf[R][KS];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = rt * ROWS + r * kRowTile + col;  // the lane's row
    const int qi = row / a.group, head = kvh * a.group + row % a.group;
    sees[r] = a.causal ? max(0, length - a.queries + 1 + qi) : length;
    const T* qrow = (const T*)a.q + b * a.qs[0] + query_at(a, qi) + head * a.qs[2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[r][s] = row < a.rows ? load_q<T, SRC != kSrcAny>(qrow, Tile::q_channel(s, g), a.d) : zero_frag<T>();
  }
  if (a.causal) {
    const int last = min(rt * ROWS + ROWS - 1, a.rows - 1) / a.group;
    all_see = max(0, length - a.queries + 1 + rt * ROWS / a.group);
    visible = max(0, min(length, length - a.queries + 1 + last));
  }
  part_of(a, length, visible, split, STEP, begin, end);

  P* vt = reinterpret_cast<P*>(lds) + wave * kKeyTile * STRIDE;
  v4f acc[R][DT];
  float m[R], l[R];
  bool seen[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
    m[r] = -INFINITY;
    l[r] = 0.f;
    seen[r] = false;
  }
  const T* kbase = (const T*)a.k + b * a.ks[0] + kvh * a.ks[2];
  const T* vbase = (const T*)a.v + b * a.vs[0] + kvh * a.vs[2];

  int key0 = begin + wave * kKeyTile;
  if (key0 < end) {
    Tile tile;
    tile.keys = know_tile<SRC, kKeyTile>(a, ask_tile<SRC, kKeyTile>(a, b, key0, lane), kvh, key0, end, lane);
    tile.load(a, kbase, vbase, kvh, key0, begin, lane);
    TileAsk ask = ask_tile<SRC, kKeyTile>(a, b, key0 + STEP, lane);
    for (; key0 < end; key0 += STEP) {
      const TileKeys keys = tile.keys;
      v4f s[R][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const FT kf = tile.k_frag(t, i);
#pragma unroll
          for (int r = 0; r < R; ++r) s[r][t] = mma16(kf, qf[r][i], s[r][t]);
        }
      }
      tile.template store_v<STRIDE>(vt, lane);  // rows that do not count are 0
#pragma unroll
      for (int r = 0; r < R; ++r) settle(s[r][0], s[r][1]);
      // the next tile (past the end: nothing counts, nothing is read)
      tile.keys = know_tile<SRC, kKeyTile>(a, ask, kvh, key0 + STEP, end, lane);
      tile.load(a, kbase, vbase, kvh, min(key0 + STEP, a.keys), begin, lane);
      ask = ask_tile<SRC, kKeyTile>(a, b, min(key0 + 2 * STEP, a.keys), lane);

      FP pf[R][Second<T, SRC>::parts];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        // scores in units of ln 2 (over the cache with the page's scale)
        float x[8], top = -INFINITY;
        float vscale[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float c = SRC == kSrcInt8 ? a.scale_log2 * lane_float(keys.kscale, t * 16) : a.scale_log2;
          vscale[t] = SRC == kSrcInt8 ? lane_float(keys.vscale, t * 16) : 1.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) x[t * 4 + j] = s[r][t][j] * c;
        }
        if ((uint32_t)keys.counts == 0xffffffffu && key0 + kKeyTile <= all_see) {  // uniform
          seen[r] = true;
        } else {
          const int n = min(max(sees[r] - key0, 0), kKeyTile);
          const uint32_t on = (uint32_t)keys.counts & (uint32_t)((1ull << n) - 1), mine = on >> (4 * g);
          seen[r] |= on != 0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(mine >> ((i >> 2) * 16 + (i & 3)) & 1)) x[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, x[i]);
        top = max32(max16(top));
        if (__any(top > m[r] + kRoom<P>)) {
          const float to = fmaxf(m[r], top - kBelow<P>);
          const float keep = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - to);
          m[r] = to;
          l[r] *= keep;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][t][i] *= keep;
        }
        const float base = m[r] == -INFINITY ? 0.f : m[r];  // nothing seen yet, or only scores of -infinity
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float p = __builtin_amdgcn_exp2f(x[i] - base);
          l[r] += p;
          if constexpr (SRC == kSrcInt8) p *= vscale[i >> 2];
          pf[r][0][i] = (P)p;
          if constexpr (Second<T, SRC>::parts == 2) pf[r][1][i] = (P)(p - (float)pf[r][0][i]);
        }
      }
      // the wave's LDS operations are in order; the compiler keeps them so
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const FP vf = load_v16<P, STRIDE>(vt, t * 16, lane);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int i = 0; i < Second<T, SRC>::parts; ++i) acc[r][t] = mma16(vf, pf[r][i], acc[r][t]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int t = 0; t < DT; ++t) settle(acc[r][t]);
  }

#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] += __shfl_xor(l[r], 16);
    l[r] += __shfl_xor(l[r], 32);
    int any = seen[r];
    any |= __shfl_xor(any, 16);
    any |= __shfl_xor(any, 32);
    if (l[r] != l[r]) m[r] = INFINITY;                     // NaN to whoever joins this
    else if (m[r] == -INFINITY) l[r] = any ? -1.f : 0.f;  // scores of -infinity alone: 0 / 0, told from a row that sees nothing

    // join the waves
    __syncthreads();
    constexpr int OS = DP + 4;
    float* mo = reinterpret_cast<float*>(lds);                            // [waves][16][OS]
    float2* ml = reinterpret_cast<float2*>(mo + kWaves * kRowTile * OS);  // [waves][16]
#pragma unroll
    for (int t = 0; t < DT; ++t) *reinterpret_cast<v4f*>(mo + (wave * kRowTile + col) * OS + t * 16 + 4 * g) = acc[r][t];
    if (g == 0) ml[wave * kRowTile + col] = make_float2(m[r], l[r]);
    __syncthreads();
    for (int i = wave * (kRowTile / kWaves); i < (wave + 1) * (kRowTile / kWaves); ++i)
      join_waves<T, OS>(a, mo, ml, i, rt * ROWS + r * kRowTile + i, b, kvh, split, lane);
  }
}

template <class T, int DP, int SRC>
__global__ __launch_bounds__(kWaves * 64, rows_per_cu(sizeof(T), DP, SRC)) void attn_rows_kernel(AttnArgs a) {
  extern __shared__ char lds[];
  rows_body<T, DP, SRC>(a, blockIdx.x, lds);
}

// Joins parts of one row's result for V of its channels: part i's maximum and
// sum at ml(i), its sums at o(i).
template <class T, int V, class ML, class O>
__device__ __forceinline__ void join_parts(int parts, ML ml, O o, T* out) {
  typedef float VF __attribute__((ext_vector_type(V)));
  float top = -INFINITY, total = 0.f, sum[V] = {};
  bool nan = false;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float2 p = ml(i);
    const VF x = *reinterpret_cast<const VF*>(o(i));
    nan |= p.y < 0.f;
    const float to = fmaxf(top, p.x);
    // -infinity: a part without a score above it has no weight
    const float keep = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - to);
    const float w = p.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(p.x - to);
    total = total * keep + (p.x == -INFINITY ? 0.f : w * p.y);
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = sum[j] * keep + (p.x == -INFINITY ? 0.f : w * x[j]);
    top = to;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = top == -INFINITY ? (nan ? NAN : 0.f) : sum[j] / total;
  Vec<T, V>::store(out, sum);
}

template <class T, int V>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int cols = a.d / V, c = (int)(item % cols) * V;
  const int64_t prow = item / cols;
  if (prow >= (int64_t)a.batch * a.kv_heads * a.rows) return;
  const int row = (int)(prow % a.rows);
  const int64_t bk = prow / a.rows;
  const int kvh = (int)(bk % a.kv_heads);
  const int64_t b = bk / a.kv_heads;
  join_parts<T, V>(
      a.splits, [&](int i) { return a.part_ml[prow * a.splits + i]; },
      [&](int i) { return a.part_o + (prow * a.splits + i) * a.d + c; },
      (T*)a.o + ((b * a.queries + row / a.group) * a.heads + kvh * a.group + row % a.group) * a.d + c);
}

template <class T, int DP, int SRC>
int rows_launch(const AttnArgs& a, hipStream_t s) {
  constexpr int bytes = rows_lds<T, DP, SRC>();
  if (bytes > 65536) NHIP_TRY(ensure_dynamic_lds((const void*)attn_rows_kernel<T, DP, SRC>, bytes));
  const uint32_t wgs = (uint32_t)((int64_t)a.batch * a.kv_heads * a.splits * a.row_tiles);
  NHIP_LAUNCH("attention_rows", (attn_rows_kernel<T, DP, SRC>), dim3(wgs), dim3(kWaves * 64), bytes, s, a);
  return check_launch("attention_rows");
}

}  // namespace attn
}  // namespace nhip

#include "attn_tiles.h"

namespace nhip {
namespace attn {

template <class T, int DP, int SRC>
int launch(const AttnArgs& a, hipStream_t s) {
  if constexpr (SRC != kSrcAny) {
    if (a.tiles) return tiles_launch<T, DP, SRC>(a, s);
  }
  return rows_launch<T, DP, SRC>(a, s);
}

template <class T, int SRC>
int launch_by_dim(const AttnArgs& a, hipStream_t s) {
  if (a.d <= 64) return launch<T, 64, SRC>(a, s);
  if (a.d <= 128) return launch<T, 128, SRC>(a, s);
  return launch<T, 256, SRC>(a, s);
}

template <class T>
int run(const AttnArgs& a, int src, hipStream_t s) {
  const int st = src == kSrcVec   ? launch_by_dim<T, kSrcVec>(a, s)
                 : src == kSrcAny ? launch_by_dim<T, kSrcAny>(a, s)
                                  : launch_by_dim<T, kSrcInt8>(a, s);
  NHIP_TRY(st);
  if (a.tiles || a.splits == 1) return ok();
  const int64_t rows = (int64_t)a.batch * a.kv_heads * a.rows;
  if (a.d % 4 == 0 && aligned_to(a.o, 4 * sizeof(T)))
    NHIP_LAUNCH("attention_join", (attn_join_kernel<T, 4>), dim3((uint32_t)ceil_div(rows * (a.d / 4), 256)), dim3(256), 0, s, a);
  else
    NHIP_LAUNCH("attention_join", (attn_join_kernel<T, 1>), dim3((uint32_t)ceil_div(rows * a.d, 256)), dim3(256), 0, s, a);
  return check_launch("attention_join");
}

// Where the parts of a row lie: of batch b's key/value head kvh.
struct RowParts {
  int count;
  int64_t first, step;  // places of the parts
  __device__ __forceinline__ RowParts(const AttnArgs& a, int b, int kvh, int row) {
    const int64_t head = (int64_t)b * a.kv_heads + kvh;
    if (a.tiles) {
      const uint32_t tile = (uint32_t)(head * a.row_tiles + row / kTilesRows);
      const bool dealt = a.workers != a.batch * a.kv_heads * a.row_tiles;
      const int worker = dealt ? worker_of(a, tile * a.units) : (int)tile;
      count = dealt ? worker_of(a, (tile + 1) * a.units - 1) - worker + 1 : 1;
      first = ((int64_t)worker + tile) * kTilesRows + row % kTilesRows;
      step = kTilesRows;
    } else {
      count = a.splits;
      first = (head * a.rows + row) * a.splits;
      step = 1;
    }
  }
  __device__ __forceinline__ int64_t place(int i) const { return first + i * step; }
};

// Joins the parts of a row's keys in the prefix and of its own, four channels to a
// thread: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i.  Bytes bound it, most of them
// still in the last-level cache: 48 sequences of 28 rows, 8 heads of 128 10.4 us.
template <class T>
__global__ __launch_bounds__(256) void attn_prefix_join_kernel(AttnArgs prefix, AttnArgs a) {
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int cols = a.d / 4, c = (int)(item % cols) * 4;
  const int64_t prow = item / cols;
  if (prow >= (int64_t)a.batch * a.kv_heads * a.rows) return;
  const int row = (int)(prow % a.rows), kvh = (int)(prow / a.rows % a.kv_heads), b = (int)(prow / a.rows / a.kv_heads);
  const int members = a.batch / prefix.batch;
  const RowParts shared(prefix, b / members, kvh, b % members * a.rows + row), own(a, b, kvh, row);
  join_parts<T, 4>(
      shared.count + own.count,
      [&](int i) { return i < shared.count ? prefix.part_ml[shared.place(i)] : a.part_ml[own.place(i - shared.count)]; },
      [&](int i) {
        return (i < shared.count ? prefix.part_o + shared.place(i) * a.d : a.part_o + own.place(i - shared.count) * a.d) + c;
      },
      (T*)a.o + (((int64_t)b * a.queries + row / a.group) * a.heads + kvh * a.group + row % a.group) * a.d + c);
}

// Both parts in one launch: the sequences' own keys, few rows each, and then the
// prefix, whose rows are those of a whole group of sequences, so that its keys are
// read and converted once for all of them.  Each workgroup is one of the kernels above, and its
// result a part; one launch because either alone leaves CUs idle (one group of 5
// sequences, 12 heads of 64, 197 and 37 keys fp32 20.4 us a call in two, 14.1 in one, the prefix whole; 48
// of 28 rows, 12544 and 1568 keys 211 and 185).  The products and the codes' conversion
// bound it where a group has many rows (the latter 165 us without the join, fp16, 8 heads
// of 128), waits for loads where it has few (4 groups of 64 rows, 3136 and 256 keys,
// bf16 34 us; 51 MB read, 124 past the L2s: the dies' own or one's, the time is the same;
// with the prefix first 2 us more).  All results pass through memory as fp32 parts and a
// join, which pays where many sequences of few queries share a long prefix.  us, so / the
// attention over one table of both, 32 heads on 8 of 128 bf16, one group, causal, as many
// own keys as queries: 64 sequences of 1 query behind 197 / 3136 / 12544 keys 28 / 14, 40 / 62,
// 49 / 195, of 4 32 / 15, 51 / 66, 96 / 199, of 16 58 / 23, 147 / 140, 312 / 524, of 32 63 / 27, 179
// / 145, 568 / 535; 16 of 1 16 / 12, 21 / 27, 39 / 58, of 16 26 / 15, 51 / 51, 97 / 146; 4 of 1 17 /
// 12, 18 / 18, 24 / 29; prompts of 4 x 512 behind 197 and 3136 81 / 44 and 197 / 163, of 16 x 1024
// 596 / 355 and 1513 / 1289.  OWN == 2 has too many registers for as many workgroups to a CU.
template <class T, int DP, bool TILES, int OWN>
__global__ __launch_bounds__(kWaves * 64, (TILES ? TilesShape<T, DP, kSrcInt8>::per_cu : rows_per_cu(sizeof(T), DP, kSrcInt8) - (OWN == 2 && DP == 128 && sizeof(T) == 2))) void
attn_prefix_kernel(AttnArgs prefix, AttnArgs own, uint32_t own_wgs) {
  extern __shared__ char lds[];
  if (blockIdx.x < own_wgs)
    rows_body<T, DP, kSrcInt8, OWN>(own, blockIdx.x, lds);
  else if constexpr (TILES)
    tiles_body<T, DP, kSrcInt8>(prefix, blockIdx.x - own_wgs, gridDim.x - own_wgs, lds);
  else
    rows_body<T, DP, kSrcInt8>(prefix, blockIdx.x - own_wgs, lds);
}

template <class T, int DP, bool TILES, int OWN>
int prefix_launch(const AttnArgs& prefix, const AttnArgs& own, hipStream_t s) {
  constexpr int rows = rows_lds<T, DP, kSrcInt8>(), tiles = TilesShape<T, DP, kSrcInt8>::bytes;
  constexpr int bytes = TILES && tiles > rows ? tiles : rows;
  if (bytes > 65536) NHIP_TRY(ensure_dynamic_lds((const void*)attn_prefix_kernel<T, DP, TILES, OWN>, bytes));
  const int64_t own_wgs = (int64_t)own.batch * own.kv_heads * own.splits * own.row_tiles;
  const int64_t wgs = TILES ? ceil_div(prefix.workers, 8) * 8 : (int64_t)prefix.batch * prefix.kv_heads * prefix.splits * prefix.row_tiles;
  NHIP_LAUNCH("attention_prefix", (attn_prefix_kernel<T, DP, TILES, OWN>), dim3((uint32_t)(own_wgs + wgs)), dim3(kWaves * 64), bytes, s,
              prefix, own, (uint32_t)own_wgs);
  return check_launch("attention_prefix");
}

template <class T, int DP>
int prefix_parts(const AttnArgs& prefix, const AttnArgs& own, hipStream_t s) {
  if (!own.tiles) {
    if constexpr (DP <= 128)
      if (own.reps == 2) return prefix.tiles ? prefix_launch<T, DP, true, 2>(prefix, own, s) : prefix_launch<T, DP, false, 2>(prefix, own, s);
    return prefix.tiles ? prefix_launch<T, DP, true, 1>(prefix, own, s) : prefix_launch<T, DP, false, 1>(prefix, own, s);
  }
  NHIP_TRY((launch<T, DP, kSrcInt8>(prefix, s)));
  return launch<T, DP, kSrcInt8>(own, s);
}

template <class T>
int run_prefix(const AttnArgs& prefix, const AttnArgs& a, hipStream_t s) {
  NHIP_TRY(a.d <= 64 ? (prefix_parts<T, 64>(prefix, a, s)) : a.d <= 128 ? (prefix_parts<T, 128>(prefix, a, s)) : (prefix_parts<T, 256>(prefix, a, s)));
  const int64_t items = (int64_t)a.batch * a.kv_heads * a.rows * (a.d / 4);
  NHIP_LAUNCH("attention_prefix_join", (attn_prefix_join_kernel<T>), dim3((uint32_t)ceil_div(items, 256)), dim3(256), 0, s, prefix, a);
  return check_launch("attention_prefix_join");
}

}  // namespace attn
}  // namespace nhip
