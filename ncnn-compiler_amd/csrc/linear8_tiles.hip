// Products in 8-bit integers for many rows: tiles of 128 rows and 256 channels,
// and quarters of them where few are left over.
#include <algorithm>
#include <type_traits>

#include "lds_dma.h"
#include "linear8.h"

namespace nhip {
namespace {

constexpr int kWaves = 4, kSlots = 3;  // stages that LDS holds

// A workgroup's tile: its waves are two by two, each has 32 CB channels, 32 RB rows.
template <int CB, int RB>
struct Tile {
  static constexpr int kCols = 64 * CB, kRows = 64 * RB;
  static constexpr int kStage = (kRows + kCols) * kStepK;  // bytes: the weights' steps, then the tokens'
  template <class T>
  static constexpr int stride = 32 * CB + kVec<T>;  // of the results' rows in LDS: those written together lie in different banks
  template <class T>
  static constexpr int lds() {
    constexpr int out = 2 * kCols * (int)sizeof(float) + kWaves * 32 * stride<T> * (int)sizeof(T);
    return std::max(kSlots * kStage, out);
  }
};
typedef Tile<4, 2> Large;
typedef Tile<2, 1> Small;  // a quarter of it
constexpr int kRows = Large::kRows;
// Row tiles that are taken together (below).  us a call at 1 / 2 / 8: 6272 x 8192 of 2048
// bf16 148 / 121 / 117, 8192 x 8192 of 8192 657 / 509 / 504, 2048 x 8192 of 4096 91 / 74 / 74;
// 4 and 16 as 8.
constexpr int kGroup = 8;

// The expert and its row tile that tile `at` of all row tiles is: experts
// without rows have none.  All 64 lanes call it.
__device__ __forceinline__ bool find_tile(const Linear8Args& a, int at, int& e, int& begin, int& end) {
  e = 0;
  expert_rows(a, 0, begin, end);
  if (!a.starts) {
    begin += at * kRows;
    return begin < end;
  }
  const int lane = threadIdx.x & 63;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    int b = 0, t = 0;
    if (e0 + lane < a.experts) expert_rows(a, e0 + lane, b, t);
    const int tiles = (t - b + kRows - 1) / kRows;
    int upto = tiles;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int v = __shfl_up(upto, o);
      if (lane >= o) upto += v;
    }
    const uint64_t past = __ballot(at < upto);
    if (past) {
      const int l = __builtin_ctzll(past);
      e = e0 + l;
      begin = __builtin_amdgcn_readlane(b, l) + (at - __builtin_amdgcn_readlane(upto - tiles, l)) * kRows;
      end = __builtin_amdgcn_readlane(t, l);
      return true;
    }
    at -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

__device__ __forceinline__ int round_up8(int v) { return (v + 7) & ~7; }

// f of the whole numbers below N, as constants.
template <int N, class F, int I = 0>
__device__ __forceinline__ void each(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>());
    each<N, F, I + 1>(f);
  }
}

// STREAM: results past kStreamBytes take no place in the caches: 6272 x 8192 of
// 2048 bf16 111 -> 106 us, 12544 x 4096 of 1024 fp16 117 -> 109.
template <bool STREAM>
__device__ __forceinline__ void store16(void* to, const void* from) {
  const v4i v = *reinterpret_cast<const v4i*>(from);
  if constexpr (STREAM)
    __builtin_nontemporal_store(v, reinterpret_cast<v4i*>(to));
  else
    *reinterpret_cast<v4i*>(to) = v;
}

// Rows begin .. end - 1 (at most SHAPE::kRows count) and channels from block b0 of expert e.
template <class SHAPE, int CB, int RB, class T, int ACT, bool STREAM>
__device__ __forceinline__ void tile_body(const Linear8Args& a, int e, int begin, int end, int b0, char* lds) {
  constexpr int kCols = SHAPE::kCols, kRows = SHAPE::kRows, kStage = SHAPE::kStage;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;

  // A wave's copies of a stage, 1 KB each.
  constexpr int WCOPIES = kCols / 16 / kWaves, XCOPIES = kRows / 16 / kWaves, COPIES = WCOPIES + XCOPIES;
  const v4i wrsrc = dma::raw_rsrc(a.w + ((int64_t)e * a.blocks + b0) * a.steps * 1024, 0x7fffffffu);
  const v4i xrsrc = dma::raw_rsrc(a.x + (int64_t)(begin >> 4) * a.steps * 1024, 0x7fffffffu);
  uint32_t woff[WCOPIES], xoff[XCOPIES];
#pragma unroll
  for (int i = 0; i < WCOPIES; ++i)
    woff[i] = (uint32_t)(min(wave * WCOPIES + i, a.blocks - 1 - b0) * a.steps) * 1024u + lane * 16;
#pragma unroll
  for (int i = 0; i < XCOPIES; ++i) {
    const int row = min((wave * XCOPIES + i) * 16 + (lane & 15), end - 1 - begin);
    xoff[i] = (uint32_t)code_at((begin & 15) + row, a.steps) + (lane >> 4) * 256;
  }
  // (past the last stage nothing is read, and zeros are written)
  const auto copy = [&](int stage, int slot, auto i) {
    v4i rsrc = i < WCOPIES ? wrsrc : xrsrc;
    rsrc[2] = stage < a.steps ? 0x7fffffff : 0;
    const uint32_t to = lds0 + slot * kStage;
    if constexpr (i < WCOPIES)
      dma::copy16(to + (wave * WCOPIES + i) * 1024, woff[i], rsrc, stage * 1024u);
    else
      dma::copy16(to + (kCols / 16 + wave * XCOPIES + i - WCOPIES) * 1024, xoff[i - WCOPIES], rsrc, stage * 1024u);
  };
  const int wc = wave & 1, wr = wave >> 1;
  // what the results need: a thread's channel's scale and bias, its rows' scales
  static_assert(kWaves * 64 >= kCols, "a thread to each channel");
  const int channel = b0 * 16 + threadIdx.x;
  const float w_scale = channel < a.n ? a.w_scale[(int64_t)e * a.n + channel] : 0.f;
  const float w_bias = channel < a.n ? a.bias[(int64_t)e * a.n + channel] : 0.f;
  float xs[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) xs[r] = a.x_scale[min(begin + (wr * RB + r) * 32 + (lane & 31), end - 1)];
  v16i acc[CB][RB];
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][r][i] = 0;
  // lane's 16 codes of a 32 x 32 block: row lane & 31, codes 16 (lane >> 5) ..
  const uint32_t lane_at = ((lane >> 4) & 1) * 1024u + (lane >> 5) * 256u + (lane & 15) * 16u;
  struct Step {
    v4i w[CB], x[RB];
  } step[2];
  const auto read = [&](int slot, int k, Step& f) {
    const char* at = lds + slot * kStage + lane_at + k * 512;
#pragma unroll
    for (int i = 0; i < CB; ++i) f.w[i] = *reinterpret_cast<const v4i*>(at + (wc * CB + i) * 2048);
#pragma unroll
    for (int i = 0; i < RB; ++i) f.x[i] = *reinterpret_cast<const v4i*>(at + kCols * kStepK + (wr * RB + i) * 2048);
  };
  const auto product = [&](const Step& f, auto n) {
    constexpr int c = n / RB, r = n % RB;
    acc[c][r] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[c], f.x[r], acc[c][r], 0, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
  // One barrier a stage, before its last products, whose operands are in
  // registers by then: behind it the stage's place in LDS is free for the stage
  // kSlots further on, and the next one is whole, so that its first operands and
  // the copies are under way during those products.  A copy goes between two
  // products: all at once would hold the products up.
  const int stages = a.steps;
  for (int st = 0; st < kSlots; ++st) each<COPIES>([&](auto i) { copy(st, st, i); });
  dma::wait_vmcnt<(kSlots - 1) * COPIES>();
  __builtin_amdgcn_s_barrier();
  read(0, 0, step[0]);
  int slot = 0;
  for (int st = 0; st < stages; ++st) {
    const int next = slot + 1 == kSlots ? 0 : slot + 1;
    read(slot, 1, step[1]);
    __builtin_amdgcn_sched_barrier(0);
    each<CB * RB>([&](auto n) { product(step[0], n); });
    dma::wait_vmcnt<(kSlots - 2) * COPIES>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(next, 0, step[0]);  // (past the last stage: not used)
    __builtin_amdgcn_sched_barrier(0);
    each<std::max(CB * RB, COPIES)>([&](auto n) {
      if constexpr (n < CB * RB) product(step[1], n);
      if constexpr (n < COPIES) copy(st + kSlots, slot, n);
      __builtin_amdgcn_sched_barrier(0);
    });
    slot = next;
  }
  dma::wait_vmcnt<0>();
  // (settle8 for all of them, where they are)
  asm volatile("s_nop 15\n\ts_nop 15");
#pragma unroll
  for (int c = 0; c < CB; ++c)
#pragma unroll
    for (int r = 0; r < RB; ++r) asm volatile("" : "+a"(acc[c][r]));
  __syncthreads();

  // The results through LDS, 32 rows of a wave's channels at a time, so that whole
  // rows are stored.  A lane has row lane & 31, channels 8 (i / 4) + 4 (lane >> 5) + i % 4.
  constexpr int V = kVec<T>, STRIDE = SHAPE::template stride<T>, WIDE = 32 * CB;
  T* stage = reinterpret_cast<T*>(lds + 2 * kCols * sizeof(float)) + wave * 32 * STRIDE;
  float* const params = reinterpret_cast<float*>(lds);  // [2][kCols]
  if (threadIdx.x < kCols) {
    params[threadIdx.x] = w_scale;
    params[kCols + threadIdx.x] = w_bias;
  }
  __syncthreads();
  const bool vec = a.n % V == 0 && ((uintptr_t)a.out & 15) == 0;
  const int j0 = b0 * 16 + wc * WIDE, width = min(WIDE, a.n - j0);
#pragma unroll
  for (int r = 0; r < RB; ++r) {
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int j = c * 32 + (i >> 2) * 8 + (lane >> 5) * 4;
        const v4f ws = *reinterpret_cast<const v4f*>(params + wc * WIDE + j);
        const v4f bias = *reinterpret_cast<const v4f*>(params + kCols + wc * WIDE + j);
        float y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = finish8<ACT>(acc[c][r][i + u], xs[r], ws[u], bias[u]);
        Vec<T, 4>::store(stage + (lane & 31) * STRIDE + j, y);
      }
    // the wave's LDS operations are in order; the compiler keeps them so
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int row0 = begin + (wr * RB + r) * 32, rows = min(32, end - row0);
    T* out = (T*)a.out + (int64_t)row0 * a.n + j0;
    if (vec) {
      constexpr int PER = WIDE / V;  // vectors of a row
      const int c = lane % PER * V;
#pragma unroll
      for (int i = 0; i < 32; i += 64 / PER) {
        const int at = i + lane / PER;
        if (at < rows && c < width)
          store16<STREAM>(out + (int64_t)at * a.n + c, stage + at * STRIDE + c);
      }
    } else {
      for (int i = 0; i < rows; ++i)
#pragma unroll
        for (int c = lane; c < WIDE; c += 64)
          if (c < width) out[(int64_t)i * a.n + c] = stage[i * STRIDE + c];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// Quarters of the first `small` tiles, then the other tiles whole.
// 8192 x 8192 of 8192 504 us with the codes (2180 TOPS; the library's product 2068), 6272 x
// 8192 of 2048 bf16 107 us without (1970; 1647). Of the latter the matrix units are busy 46%;
// waits for stages and barriers stand beside them (93 us with no results stored, 115 with, each
// launch timed by itself), then the results' way through LDS; 12544 x 4096 of 1024, 32 experts,
// 66 and 95 so.  32 x 32 x 32 instructions ran at 4775 TOPS from registers on zeros and
// 3400 on random codes, at a clock of some 1.7 GHz, 16 x 16 x 64 ones at 2590, so
// large instructions; two workgroups of 4 waves a CU, so that one's results and starts
// are beside the other's products.
template <class T, int ACT, bool STREAM>
__global__ __launch_bounds__(kWaves * 64, 2) void linear8_tiles_kernel(Linear8Args a, int col_tiles, int work, int small) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const auto place = [&](int id, int& e, int& begin, int& end, int& b0) {
    // blocks of kGroup row tiles, so that what a die's CUs work on at a time are
    // few row tiles and few column tiles, which meet in its L2
    const int band = id / (kGroup * col_tiles), in = id - band * kGroup * col_tiles;
    const int high = min(kGroup, work / col_tiles - band * kGroup);
    const int col = in / high;
    b0 = col * (Large::kCols / 16);
    return find_tile(a, band * kGroup + in - col * high, e, begin, end);
  };
  // workgroups go to the eight dies in turn: each die gets a run of the tiles
  const auto run = [](int block, int blocks) { return (block & 7) * (blocks >> 3) + (block >> 3); };
  const int smalls = round_up8(4 * small);
  int e, begin, end, b0;
  if ((int)blockIdx.x >= smalls) {
    const int id = small + run(blockIdx.x - smalls, gridDim.x - smalls);
    if (id >= work || !place(id, e, begin, end, b0)) return;
    tile_body<Large, 4, 2, T, ACT, STREAM>(a, e, begin, end, b0, lds);
  } else {
    const int id = run(blockIdx.x, smalls);
    if (id >= 4 * small || !place(id >> 2, e, begin, end, b0)) return;
    begin += (id & 1) * Small::kRows;
    b0 += (id >> 1 & 1) * (Small::kCols / 16);
    if (begin >= end || b0 >= a.blocks) return;
    tile_body<Small, 2, 1, T, ACT, STREAM>(a, e, begin, min(end, begin + Small::kRows), b0, lds);
  }
}

template <class T, int ACT, bool STREAM>
int tiles_launch(const Linear8Args& a, hipStream_t s) {
  constexpr int bytes = Large::lds<T>();
  static_assert(bytes <= 80 * 1024 && Small::lds<T>() <= bytes, "two workgroups a CU");
  NHIP_TRY(ensure_dynamic_lds((const void*)linear8_tiles_kernel<T, ACT, STREAM>, bytes));
  const int64_t cols = ceil_div(a.blocks, Large::kCols / 16);
  // every expert's last tile may be a part of one
  const int64_t rows = ceil_div(a.rows, kRows) + (a.starts ? std::min(a.experts, a.rows) : 0);
  if (rows * cols > 0xff0000) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "linear8: too many tiles");
  const int64_t work = rows * cols;
  const int64_t places = 2 * cu_count(), over = a.starts ? 0 : work % places;
  // A round of the CUs' places that whole tiles would fill to a quarter or less takes
  // about a quarter of its time so: 6272 x 8192 of 2048 bf16 (1568 tiles on 512 places) 125.6 us
  // without, 120.7 with.  Where sums are short, storing takes a good part of a tile's time, and
  // the places all store at once unless some begin with a part: without / with an eighth of
  // the places' number 6272 x 4096 of 1024 52.8 / 46.7, 12544 x 4096 of 1024, 32 experts 108.2 /
  // 103.5, 6000 x 4096 of 512 34.8 / 33.8; not in longer ones, 25088 x 2048 of 2048 133 / 133,
  // 6272 x 8192 of 2048 120.9 / 122.7, nor in one round, 12544 x 1024 of 2048 52.9 / 59.2.
  // Few tiles in all, each expert's counted with a part of one: quarters for every one, 3356
  // rows of 5792 over 20 experts to 320 fp32 (94 tiles) 38.3 / 27.2, 2000 of 1024 over 8 to 1024
  // bf16 14.1 / 11.0; not for more than a quarter of the places, 3000 x 1500 of 8192 54 / 67.
  int64_t small = work * 4 <= places ? work : over * 4 <= places ? over : 0;
  if (work > places && a.steps <= 16) small = std::max(small, places / 8);
  const int64_t large = work - small;
  NHIP_LAUNCH("linear8_tiles", (linear8_tiles_kernel<T, ACT, STREAM>), dim3((uint32_t)(round_up(4 * small, 8) + round_up(large, 8))), dim3(kWaves * 64),
              bytes, s, a, (int)cols, (int)work, (int)small);
  return check_launch("linear8_tiles");
}

template <class T, int ACT>
int tiles_run(const Linear8Args& a, hipStream_t s) {
  return (int64_t)a.rows * a.n * (int64_t)sizeof(T) > kStreamBytes ? tiles_launch<T, ACT, true>(a, s) : tiles_launch<T, ACT, false>(a, s);
}

}  // namespace

bool linear8_tiles_selected(const Linear8Args& a) {
  const int force = setting_int("NHIP_LINEAR8_TILES", -1);
  if (force >= 0) return force != 0;
  // Few tiles leave CUs idle and each walks the whole sum alone; the other kernel has
  // a workgroup for 64 rows and 16 channels, whose waves share the sum, and reads
  // the operands more often.  us, it / this, bf16: 300 x 1000 of 8192 (40 quarter tiles) 18.6 /
  // 27.6, 600 x 1000 (80) 23.1 / 30.6, 1200 x 1000 (152) 28.6 / 31.5, 2400 x 528 (190) 35.8 /
  // 30.1; of 3600 15.0 / 17.1 (80), 18.8 / 17.7 (152), 21.6 / 17.5 (190); of 1024 7.7 / 8.8 (40),
  // 9.4 / 9.1 (80), 11.3 / 9.1 (152), 12.4 / 9.5 (190).
  return a.rows > 64 * (int64_t)a.experts && ceil_div(a.rows, Small::kRows) * ceil_div(a.blocks, Small::kCols / 16) > cu_count() / 2;
}

int linear8_tiles(const Linear8Args& a, int dtype, hipStream_t s) {
  return NHIP_FOR_ELEM(dtype, T, NHIP_FOR_ACT(a.act, ACT, tiles_run<T, ACT>(a, s)));
}

}  // namespace nhip
