// Attention of many query rows: 128 rows to a workgroup, 32 to a wave, tiles
// of keys and values staged in LDS for all of them.  (Included by attention.h.)

namespace nhip {
namespace attn {

// Page scales of values below this add nothing to an fp16 result.
constexpr float kLeastUnit = 0x1p-60f, kMostUnit = 0x1p60f;

// fp32 values as sums of bf16 pieces, largest first: x = hi + mid + lo exactly
// (each rounding leaves at most 16, then 8 significant bits) while lo is above
// bf16's smallest normal number and hi below its largest.  A product of two
// such sums without the products of mid and lo, lo and mid, lo and lo, below
// 2^-25 of it: six matrix instructions on bf16 in place of eight on fp32 that
// take twice as long each.
constexpr float kPieceMost = 3.38e38f;
constexpr uint32_t kPieceLeast = (127 - 100) << 24;  // of 2^-100, the bits without the sign's place
__device__ __forceinline__ void split8(v8f x, v8b (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[0][i] = (bf16)x[i];
    const float r = x[i] - (float)p[0][i];
    p[1][i] = (bf16)r;
    p[2][i] = (bf16)(r - (float)p[1][i]);
  }
}
// Whether pieces would not hold some value that was shown to it.
struct PieceRange {
  float most = 0.f;
  uint32_t least = 0xffffffffu;
  __device__ __forceinline__ void show(float x) {
    most = fmaxf(most, fabsf(x));  // NaN passes: its pieces are NaN
    least = min(least, (__builtin_bit_cast(uint32_t, x) << 1) - 1u);  // 0 wraps around
  }
  __device__ __forceinline__ bool missed() const { return most > kPieceMost || least < kPieceLeast - 1u; }
};

// Sizes of the kernel for channels padded to DP.
template <class T, int DP, int SRC>
struct TilesShape {
  static constexpr bool split = sizeof(T) == 4;
  typedef typename std::conditional<split, bf16, T>::type M;  // what the matrix instructions take
  static constexpr int KP = split && SRC != kSrcInt8 ? 3 : 1;  // pieces of a key or value (codes are exact in one)
  static constexpr int QP = split ? 3 : 1;                     // of a query or probability
  // fp16 over the cache: the sums count in units of the page's scale (below)
  static constexpr bool units = SRC == kSrcInt8 && std::is_same<T, f16>::value;
  static constexpr int KT = DP == 256 || (split && DP == 128) ? 32 : 64;  // keys of a tile
  static constexpr int E = SRC == kSrcInt8 ? 16 : 16 / (int)sizeof(T);    // channels of a 16-byte load
  static constexpr int L = KT * DP / E / (kWaves * 64);                   // loads of a thread, keys and values each
  // Rows padded so that the eight rows of a 16-byte read, and the four of a
  // transposing read, lie in different banks.
  static constexpr int SK = DP + 8, SV = DP + 32;
  static constexpr int kplane = KT * SK, vplane = KT * SV;  // values of one piece
  static constexpr int buffer = KP * (kplane + vplane) * 2;
  // Pieces leave room for one buffer where two workgroups share a CU: a
  // second barrier a tile, and two words that say which tile they do not hold.
  static constexpr int buffers = KP == 3 ? 1 : 2;
  static constexpr int bytes = buffers * buffer + (KP == 3 ? 16 : 0);
  static constexpr int per_cu = split ? (DP == 64 ? 2 : 1) : DP == 64 && SRC == kSrcInt8 ? 3 : DP <= 128 ? 2 : 1;
};

// The next tile on its way, spread over the workgroup.
template <class T, int DP, int SRC>
struct TilesLoad {
  typedef TilesShape<T, DP, SRC> S;
  typedef typename S::M M;
  typedef typename Frag<M>::type FM;
  int4 k[S::L], v[S::L];
  __device__ __forceinline__ void load(const AttnArgs& a, const T* kbase, const T* vbase, const TileKeys& keys, int kvh, int key0, int wave, int lane) {
    constexpr int per = DP / S::E;
#pragma unroll
    for (int i = 0; i < S::L; ++i) {
      const int first = (wave * 64 + i * kWaves * 64) / per;  // a wave's 64 pieces lie inside 16 rows of a page
      const int at = wave * 64 + lane + i * kWaves * 64, r = at / per, c = at % per * S::E;
      const int64_t page = SRC == kSrcInt8 ? lane_page(keys, first & ~15) : 0;
      const bool on = keys.counts >> r & 1;
      const bool von = on & !(S::units && lane_float(keys.vscale, first & ~15) < kLeastUnit);
      k[i] = load_row16<T, SRC>(a, kbase, a.ks[1], a.cache.k, kvh, page, key0, r, c, on);
      v[i] = load_row16<T, SRC>(a, vbase, a.vs[1], a.cache.v, kvh, page, key0, r, c, von);
    }
  }
  // To LDS; whether pieces miss some value of this thread.
  __device__ __forceinline__ bool store(char* lds, int wave, int lane) const {
    constexpr int per = DP / S::E;
    PieceRange range;
#pragma unroll
    for (int i = 0; i < S::L; ++i) {
      const int at = wave * 64 + lane + i * kWaves * 64, r = at / per, c = at % per * S::E;
      M* kt = reinterpret_cast<M*>(lds) + r * S::SK + c;
      M* vt = reinterpret_cast<M*>(lds) + S::KP * S::kplane + r * S::SV + c;
      if constexpr (SRC == kSrcInt8) {
        *reinterpret_cast<FM*>(kt) = codes8<M>(k[i].x, k[i].y);
        *reinterpret_cast<FM*>(kt + 8) = codes8<M>(k[i].z, k[i].w);
        *reinterpret_cast<FM*>(vt) = codes8<M>(v[i].x, v[i].y);
        *reinterpret_cast<FM*>(vt + 8) = codes8<M>(v[i].z, v[i].w);
      } else if constexpr (S::split) {
        typedef bf16 v4b __attribute__((ext_vector_type(4)));
        const v4f kx = __builtin_bit_cast(v4f, k[i]), vx = __builtin_bit_cast(v4f, v[i]);
        v8f x;
        v8b p[3];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = kx[j];
          x[4 + j] = vx[j];
          range.show(kx[j]);
          range.show(vx[j]);
        }
        split8(x, p);
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          *reinterpret_cast<v4b*>(kt + j * S::kplane) = v4b{p[j][0], p[j][1], p[j][2], p[j][3]};
          *reinterpret_cast<v4b*>(vt + j * S::vplane) = v4b{p[j][4], p[j][5], p[j][6], p[j][7]};
        }
      } else {
        *reinterpret_cast<int4*>(kt) = k[i];
        *reinterpret_cast<int4*>(vt) = v[i];
      }
    }
    return S::KP == 3 && range.missed();
  }
};

// c + the product of two sums of pieces, smallest products first.
template <int KP, int QP, class F>
__device__ __forceinline__ v16f mma32_pieces(const F (&k)[KP], const F (&q)[QP], v16f c) {
#pragma unroll
  for (int n = QP - 1; n >= 0; --n)
#pragma unroll
    for (int i = 0; i < KP; ++i)
      if (n - i >= 0 && n - i < QP) c = mma32(k[i], q[n - i], c);
  return c;
}

// A lane's eight summed values down channel c0 + (l & 31) of V in LDS: keys
// 8 u + 4 h .. + 3 for u = 0, 1 (h = lane / 32), as eight of a score tile's
// sums lie in a lane.
template <class T, int STRIDE>
__device__ __forceinline__ typename Frag<T>::type load_v32(const T* tile, int c0, int lane) {
  const int h = lane >> 5, j = lane & 15;
  const T* at = tile + (4 * h + (j >> 2)) * STRIDE + c0 + (lane & 16) + (j & 3) * 4;
  typedef __attribute__((address_space(3))) v4s lds4;
  const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)at);
  const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at + 8 * STRIDE));
  return __builtin_bit_cast(typename Frag<T>::type, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// l + the sum of eight probabilities as the second product takes them (exact,
// summed in fp32), one instruction for two: fp16 over the cache, whose vector
// unit converts codes besides (71 us for a chunk, 73 with 32 additions; without
// codes to convert the additions were the faster, 700 us to 715).
__device__ __forceinline__ float sum8(v8h p, float l) {
  typedef f16 v2h __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 8; i += 2) l = __builtin_amdgcn_fdot2(v2h{p[i], p[i + 1]}, v2h{(f16)1.f, (f16)1.f}, l, false);
  return l;
}

// The work of a launch is row tiles x units (a unit: one of `units` equal parts
// of a row tile's keys; below 2^31 of them where they are dealt), dealt to the
// workers in equal runs.  With as many workers as row tiles each does one; with
// fewer or more, a run crosses row tiles or ends inside one.
__device__ __forceinline__ uint32_t first_unit(const AttnArgs& a, uint32_t worker) {
  const uint32_t work = (uint32_t)a.batch * a.kv_heads * a.row_tiles * a.units;
  return (uint32_t)((uint64_t)worker * work / (uint32_t)a.workers);
}
__device__ __forceinline__ int worker_of(const AttnArgs& a, uint32_t unit) {
  const uint32_t work = (uint32_t)a.batch * a.kv_heads * a.row_tiles * a.units;
  return (int)((((uint64_t)unit + 1) * a.workers - 1) / work);
}

// One workgroup, kTilesRows query rows of one key/value head at a time.  Scores,
// probabilities and sums stay in registers from one product to the other; while
// a tile is worked on, the next one's loads are under way, and it goes into the
// other of two LDS buffers: one barrier a tile.
//
// Measured.  bf16: 2 x 3136 rows of 16 heads of 128 to 12544 keys 703-729 us (827-858
// TFLOP/s, 21 us of it the join), 4096 rows and keys, whose row tiles fill the
// CUs evenly, 281-287 us (957-978; a library product of matrices alone 1130).  The
// rest is the softmax: vector instructions of one wave beside another's products.
// fp16 over the cache: 2 x 509 rows of 16 heads of 64 to 6272 keys 60 us: half
// the products to a score and codes to convert, so the waves' other instructions
// bound it.
// fp32: 4 x 784 rows of 12 heads of 64 to 197 keys 32 us, of which 12 pass before
// the first tile and after the last, and of a wave's time some 6 are vector
// instructions, 3 matrix ones; 2 x 2048 of 16 to 4096 keys 380-390 us (180
// TFLOP/s; the fp32 instructions' rate is 154), some 1000 vector instructions
// of a wave, most of them splitting, beside 96 products a tile.
template <class T, int DP, int SRC>
__global__ __launch_bounds__(kWaves * 64, (TilesShape<T, DP, SRC>::per_cu)) void attn_tiles_kernel(AttnArgs a) {
  typedef TilesShape<T, DP, SRC> S;
  typedef typename S::M M;
  typedef typename Frag<M>::type FM;
  constexpr int KT = S::KT, NT = KT / 32, KS = DP / 16, DT = DP / 32, KP = S::KP, QP = S::QP;
  constexpr int AHEAD = S::split ? 1 : KS < 8 ? KS : 8;  // operands read ahead of their products
  extern __shared__ char lds[];
  const int lane = threadIdx.x & 63, wave = wave_id(), h = lane >> 5, col = lane & 31;
  // workgroups go to the eight dies in turn: each die gets a run of workers, so
  // that those of one head meet in its L2
  const uint32_t worker = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (worker >= (uint32_t)a.workers) return;
  const bool dealt = a.workers != a.batch * a.kv_heads * a.row_tiles;
  uint32_t unit = dealt ? first_unit(a, worker) : 0, unit_end = dealt ? first_unit(a, worker + 1) : (uint32_t)a.units;
  while (unit < unit_end) {
    // units [u0, u1) of one row tile
    const uint32_t tile = dealt ? unit / (uint32_t)a.units : worker;
    const int u0 = dealt ? (int)(unit - tile * a.units) : 0, u1 = min(a.units, u0 + (int)(unit_end - unit));
    unit += u1 - u0;
    const int rt = tile % a.row_tiles, kvh = tile / a.row_tiles % a.kv_heads, b = tile / a.row_tiles / a.kv_heads;

    const int length = a.lengths ? max(0, min(a.lengths[b], a.keys)) : a.keys;
    const int row = rt * kTilesRows + wave * 32 + col;
    const int qi = row / a.group, head = kvh * a.group + row % a.group;
    int sees = length, all_see = length, visible = length;
    if (a.causal) {
      const int last = min(rt * kTilesRows + kTilesRows - 1, a.rows - 1) / a.group;
      const int first = (rt * kTilesRows + wave * 32) / a.group;
      sees = max(0, length - a.queries + 1 + qi);
      all_see = max(0, length - a.queries + 1 + first);
      visible = max(0, min(length, length - a.queries + 1 + last));
    }
    int begin = u0 * KT, end = u1 * KT;
    if (const int64_t tiles = (visible + KT - 1) / KT; tiles != a.units) {
      begin = (int)(u0 * tiles / a.units) * KT;
      end = (int)(u1 * tiles / a.units) * KT;
    }
    end = min(end, visible);

    // (pieces of more than 128 channels would not fit the registers: split at each use)
    constexpr bool LATE = S::split && DP == 256;
    FM qf[LATE ? 1 : KS][QP];
    v8f qx[LATE ? KS : 1];
    const T* qrow = (const T*)a.q + b * a.qs[0] + qi * a.qs[1] + head * a.qs[2];
    const auto query = [&](int s) {
      auto q = row < a.rows ? load_q<T, true>(qrow, s * 16 + h * 8, a.d) : zero_frag<T>();
      return a.scale_log2 < 0.f ? -q : q;
    };
    PieceRange qrange;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (S::split) {
        const v8f q = query(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) qrange.show(q[i]);
        if constexpr (LATE)
          qx[s] = q;
        else
          split8(q, qf[s]);
      } else {
        qf[s][0] = query(s);
      }
    }
    const bool qmissed = KP == 3 && __any(qrange.missed());

    v16f acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
    float m = -INFINITY, l = 0.f;
    float in = 1.f;  // what one of the sums' units stands for
    bool seen = false;
    const T* kbase = (const T*)a.k + b * a.ks[0] + kvh * a.ks[2];
    const T* vbase = (const T*)a.v + b * a.vs[0] + kvh * a.vs[2];

    if (begin < end) {
      TilesLoad<T, DP, SRC> next;
      TileKeys keys = know_tile<SRC, KT>(a, ask_tile<SRC, KT>(a, b, begin, lane), kvh, begin, end, lane);
      next.load(a, kbase, vbase, keys, kvh, begin, wave, lane);
      TileAsk ask = ask_tile<SRC, KT>(a, b, min(begin + KT, a.keys), lane);
      int* missed = reinterpret_cast<int*>(lds + S::buffers * S::buffer);  // [2], tiles by turns
      if constexpr (KP == 3) {
        if (threadIdx.x < 2) missed[threadIdx.x] = 0;
        __syncthreads();
      }
      if (__any(next.store(lds, wave, lane)) && lane == 0) missed[0] = 1;
      __syncthreads();
      int turn = 0;
      for (int key0 = begin; key0 < end; key0 += KT) {
        // the next tile (past the end: nothing counts, nothing is read)
        const int key1 = min(key0 + KT, a.keys);
        const TileKeys soon = know_tile<SRC, KT>(a, ask, kvh, key0 + KT, end, lane);
        next.load(a, kbase, vbase, soon, kvh, key1, wave, lane);
        ask = ask_tile<SRC, KT>(a, b, min(key1 + KT, a.keys), lane);

        const M* kt = reinterpret_cast<const M*>(lds + (S::buffers == 2 ? turn : 0) * S::buffer);
        const M* vt = kt + KP * S::kplane;
        const bool exact = KP == 3 && (qmissed || __builtin_amdgcn_readfirstlane(missed[turn]));
        v16f s[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[t][i] = 0.f;
        if (KP == 3 && __builtin_expect(exact, false)) {
          // values that pieces do not hold: fp32 products of the keys as they stand in memory
          if constexpr (KP == 3) {
            int kcol = col;
            asm volatile("" : "+v"(kcol));  // addresses are formed here, not kept through the loop
#pragma unroll 1
            for (int i = 0; i < KS; ++i) {
              const v8f q = query(i);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                const bool counts = keys.counts >> (t * 32 + kcol) & 1;
                struct { int4 lo, hi; } both;
                both.lo = load_row16<T, SRC>(a, kbase, a.ks[1], nullptr, 0, 0, key0, t * 32 + kcol, i * 16 + h * 8, counts);
                both.hi = load_row16<T, SRC>(a, kbase, a.ks[1], nullptr, 0, 0, key0, t * 32 + kcol, i * 16 + h * 8 + 4, counts);
                s[t] = mma32(__builtin_bit_cast(v8f, both), q, s[t]);
              }
            }
          }
        } else {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i0 = 0; i0 < KS; i0 += AHEAD) {
              FM kf[AHEAD][KP];
#pragma unroll
              for (int i = 0; i < AHEAD; ++i)
#pragma unroll
                for (int p = 0; p < KP; ++p)
                  kf[i][p] = *reinterpret_cast<const FM*>(kt + p * S::kplane + (t * 32 + col) * S::SK + (i0 + i) * 16 + h * 8);
              if constexpr (!S::split) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
              for (int i = 0; i < AHEAD; ++i) {
                if constexpr (LATE) {
                  v8b q[3];
                  split8(qx[i0 + i], q);
                  s[t] = mma32_pieces(kf[i], q, s[t]);
                } else {
                  s[t] = mma32_pieces(kf[i], qf[i0 + i], s[t]);
                }
              }
            }
        }
        if constexpr (NT == 2)
          settle(s[0], s[1]);
        else
          settle(s[0]);

        // From scores to units of ln 2, over the cache with the scale of the 16
        // keys' page; the factor goes into the exponent.  (Not 0, so that
        // -infinity stays what it is.)
        float factor[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            factor[t][u] = fmaxf(fabsf(a.scale_log2) * (SRC == kSrcInt8 ? lane_float(keys.kscale, t * 32 + u * 16) : 1.f), 1.17549435e-38f);
        constexpr uint64_t every = KT == 64 ? ~0ull : 0xffffffffull;
        const bool whole = (keys.counts & every) == every && key0 + KT <= all_see;  // uniform
        uint64_t on = every;
        if (!whole) {
          const int n = min(max(sees - key0, 0), KT);
          on = keys.counts & (n >= 64 ? ~0ull : (1ull << n) - 1);
          const uint64_t mine = on >> (4 * h);
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!(mine >> (t * 32 + (i >> 2) * 8 + (i & 3)) & 1)) s[t][i] = -INFINITY;
        }
        seen |= on != 0;
        float top = -INFINITY;
        if constexpr (SRC != kSrcInt8) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
          top *= factor[0][0];
        } else
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float most = s[t][u * 8];
#pragma unroll
            for (int i = 1; i < 8; ++i) most = fmaxf(most, s[t][u * 8 + i]);
            top = fmaxf(top, most * factor[t][u]);
          }
        top = max32(top);
        if (__any(top > m + kRoom<M>)) {
          const float to = fmaxf(m, top - kBelow<M>);
          const float keep = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
          m = to;
          l *= keep;
#pragma unroll
          for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[t][i] *= keep;
        }
        const float base = m == -INFINITY ? 0.f : m;
        // 16-bit types: probabilities are rounded to the type for the second
        // product, as with few rows.  As the sum of two they would take another one:
        // us with one / two 737 / 987 (2 x 3136 rows of 16 heads of 128 to 12544 keys
        // bf16), 23.3 / 29.7 (4 x 784 of 12 of 64 to 784), 60 / 73 (fp16 over the cache).
        // l sums them as they were; with units as rounded (sum8).
        typename std::conditional<S::split, v8f, FM>::type pf[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float vscale = SRC == kSrcInt8 && !S::units ? lane_float(keys.vscale, t * 32 + u * 16) : 1.f;
            v8f p;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][u * 8 + i], factor[t][u], -base));
              if constexpr (!S::units) l += p[i];
              if constexpr (SRC == kSrcInt8 && !S::units) p[i] *= vscale;
              if constexpr (!S::split) pf[t][u][i] = (M)p[i];
            }
            if constexpr (S::split) pf[t][u] = p;
            if constexpr (S::units) l = sum8(pf[t][u], l);
          }
        if (KP == 3 && __builtin_expect(exact, false)) {
          if constexpr (KP == 3) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int c = 0; c < DT; ++c) {
                  const __amdgpu_buffer_rsrc_t rows = make_rsrc(vbase + (int64_t)key0 * a.vs[1], 0x7fffffffu);
                  int vcol = col, vh = h;
                  asm volatile("" : "+v"(vcol), "+v"(vh));
                  v8f vf;
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    const int r = t * 32 + u * 16 + 8 * (i >> 2) + 4 * vh + (i & 3), ch = c * 32 + vcol;
                    const bool counts = (keys.counts >> r & 1) && ch < a.d;
                    vf[i] = buf_load_f32(rows, counts ? (r * (uint32_t)a.vs[1] + ch) * 4u : kBufOOB);
                  }
                  acc[c] = mma32(vf, pf[t][u], acc[c]);
                  __builtin_amdgcn_sched_barrier(0);
                }
          }
#pragma unroll
          for (int c = 0; c < DT; ++c) settle(acc[c]);
        } else {
        // (over the cache, whose other waves convert codes: 73 -> 71 us; else no gain)
        if constexpr (SRC == kSrcInt8) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if constexpr (S::units) {
              // probabilities times a page's scale may leave fp16's range, so
              // the sums change to its units instead (values of smaller ones
              // than kLeastUnit, and of pages that nobody sees, were read as 0)
              const float scale = lane_float(keys.vscale, t * 32 + u * 16), now = fminf(scale, kMostUnit);
              if (!(scale < kLeastUnit) && now != in) {
                settle(acc[0]);
                const float r = in * __builtin_amdgcn_rcpf(now);
#pragma unroll
                for (int c = 0; c < DT; ++c) {
                  asm volatile("" : "+v"(acc[c]));  // after the wait
#pragma unroll
                  for (int i = 0; i < 16; ++i) acc[c][i] *= r;
                }
                in = now;
              }
            }
            FM pp[QP];
            if constexpr (S::split)
              split8(pf[t][u], pp);
            else
              pp[0] = pf[t][u];
#pragma unroll
            for (int c = 0; c < DT; ++c) {
              FM vf[KP];
#pragma unroll
              for (int p = 0; p < KP; ++p) vf[p] = load_v32<M, S::SV>(vt + p * S::vplane + (t * 32 + u * 16) * S::SV, c * 32, lane);
              acc[c] = mma32_pieces(vf, pp, acc[c]);
            }
          }
        }
        if constexpr (SRC == kSrcInt8) __builtin_amdgcn_s_setprio(0);
        if constexpr (S::buffers == 1) {
          __syncthreads();
          if (threadIdx.x == 0) missed[turn] = 0;  // everybody has read it; next set in the tile after the next
        }
        turn ^= 1;
        if (__any(next.store(lds + (S::buffers == 2 ? turn : 0) * S::buffer, wave, lane)) && lane == 0) missed[turn] = 1;
        keys = soon;
        __syncthreads();
      }
#pragma unroll
      for (int t = 0; t < DT; ++t) settle(acc[t]);
    }
    l += __shfl_xor(l, 32);
    if (l != l) m = INFINITY;                         // NaN to whoever joins this
    else if (m == -INFINITY) l = seen ? -1.f : 0.f;  // scores of -infinity alone: 0 / 0, told from a row that sees nothing
    // a whole row tile's result, or a part: the one that begins the tile goes to
    // the worker's second place, any other to its first
    const bool whole_tile = u1 - u0 == a.units;
    const int64_t prow = ((int64_t)worker * 2 + (u0 == 0)) * kTilesRows + wave * 32 + col;
    float* part = a.part_o + prow * a.d;
    T* out = (T*)a.o + (((int64_t)b * a.queries + qi) * a.heads + head) * a.d;
    const float scale = m == -INFINITY ? (l < 0.f ? NAN : 0.f) : in / l;
    if (row < a.rows) {
      if (!whole_tile && h == 0) a.part_ml[prow] = make_float2(m, l);
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const int c = t * 32 + (i >> 2) * 8 + 4 * h;
          if (c < a.d) {
            float o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] = acc[t][i + j] * (whole_tile ? scale : in);
            if (whole_tile)
              Vec<T, 4>::store(out + c, o);
            else
              *reinterpret_cast<v4f*>(part + c) = v4f{o[0], o[1], o[2], o[3]};
          }
        }
    }
  }
}

// Joins the parts of the row tiles that several workers share.
template <class T>
__global__ __launch_bounds__(256) void attn_tiles_join_kernel(AttnArgs a) {
  const int cols = a.d / 4, per = (kTilesRows * cols + 255) / 256;  // workgroups of a row tile
  const uint32_t tile = blockIdx.x / per;
  const int w0 = worker_of(a, tile * a.units), w1 = worker_of(a, (tile + 1) * a.units - 1);
  if (w0 == w1) return;
  const int item = blockIdx.x % per * 256 + threadIdx.x, in = item / cols, c = item % cols * 4;
  const int row = tile % a.row_tiles * kTilesRows + in;
  if (in >= kTilesRows || row >= a.rows) return;
  const int kvh = tile / a.row_tiles % a.kv_heads, b = tile / a.row_tiles / a.kv_heads;
  const auto place = [&](int i) { return ((int64_t)(w0 + i) * 2 + (i == 0)) * kTilesRows + in; };
  join_parts<T, 4>(
      w1 - w0 + 1, [&](int i) { return a.part_ml[place(i)]; }, [&](int i) { return a.part_o + place(i) * a.d + c; },
      (T*)a.o + (((int64_t)b * a.queries + row / a.group) * a.heads + kvh * a.group + row % a.group) * a.d + c);
}

template <class T, int DP, int SRC>
int tiles_launch(const AttnArgs& a, hipStream_t s) {
  constexpr int bytes = TilesShape<T, DP, SRC>::bytes;
  static_assert(bytes <= 160 * 1024, "two tiles fit the LDS");
  if (bytes > 65536) NHIP_TRY(ensure_dynamic_lds((const void*)attn_tiles_kernel<T, DP, SRC>, bytes));
  NHIP_LAUNCH("attention_tiles", (attn_tiles_kernel<T, DP, SRC>), dim3((uint32_t)ceil_div(a.workers, 8) * 8),
              dim3(kWaves * 64), bytes, s, a);
  NHIP_TRY(check_launch("attention_tiles"));
  const int64_t tiles = (int64_t)a.batch * a.kv_heads * a.row_tiles;
  if (a.workers == tiles) return ok();
  NHIP_LAUNCH("attention_join", attn_tiles_join_kernel<T>, dim3((uint32_t)(tiles * ceil_div(kTilesRows * (a.d / 4), 256))),
              dim3(256), 0, s, a);
  return check_launch("attention_join");
}

}  // namespace attn
}  // namespace nhip
