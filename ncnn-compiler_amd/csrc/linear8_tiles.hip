// Products in 8-bit integers for many rows: tiles of 256 rows and 256 channels.
#include <algorithm>

#include "lds_dma.h"
#include "linear8.h"

namespace nhip {
namespace {

constexpr int kTile = 256, kWaves = 8;
constexpr int kSide = kTile * kPadK;  // bytes of one operand's stage
constexpr int kStage = 2 * kSide;
constexpr int kLds = 2 * kStage;
constexpr int kGroup = 4;

// The expert and its row tile that tile `at` of all row tiles is: experts
// without rows have none.  All 64 lanes call it.
__device__ __forceinline__ bool find_tile(const Linear8Args& a, int at, int& e, int& begin, int& end) {
  e = 0;
  expert_rows(a, 0, begin, end);
  if (!a.starts) {
    begin += at * kTile;
    return begin < end;
  }
  const int lane = threadIdx.x & 63;
  for (int e0 = 0; e0 < a.experts; e0 += 64) {
    int b = 0, t = 0;
    if (e0 + lane < a.experts) expert_rows(a, e0 + lane, b, t);
    const int tiles = (t - b + kTile - 1) / kTile;
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
      begin = __builtin_amdgcn_readlane(b, l) + (at - __builtin_amdgcn_readlane(upto - tiles, l)) * kTile;
      end = __builtin_amdgcn_readlane(t, l);
      return true;
    }
    at -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

template <class T, int ACT>
__global__ __launch_bounds__(kWaves * 64) void linear8_tiles_kernel(Linear8Args a, int col_tiles, int work) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups go to the eight dies in turn: each die gets a run of the tiles
  const int id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (id >= work) return;
  // ... in blocks of kGroup row tiles, so that what its CUs work on at a time are
  // few row tiles and few column tiles, which meet in its L2
  const int band = id / (kGroup * col_tiles), in = id - band * kGroup * col_tiles;
  const int high = min(kGroup, work / col_tiles - band * kGroup);
  const int col = in / high;
  int e, begin, end;
  if (!find_tile(a, band * kGroup + in - col * high, e, begin, end)) return;
  const int b0 = col * (kTile / 16);  // first block of channels
  const uint32_t lds0 = (uint32_t)(uintptr_t)lds;

  // A wave's copies of a stage: 4 KB of weights, 4 KB of codes, 1 KB (16 rows, 64 codes) each.
  const v4i wrsrc = dma::raw_rsrc(a.w + ((int64_t)e * a.blocks + b0) * a.steps * 1024, 0x7fffffffu);
  const v4i xrsrc = dma::raw_rsrc(a.x + (int64_t)begin * a.kp, 0x7fffffffu);
  uint32_t woff[4], xoff[4], to[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = wave * 4 + i, blk = c >> 1, half = c & 1;
    woff[i] = (uint32_t)(min(blk, a.blocks - 1 - b0) * a.steps + half) * 1024u + lane * 16;
    xoff[i] = (uint32_t)min(blk * 16 + (lane & 15), end - 1 - begin) * (uint32_t)a.kp + half * 64 + (lane >> 4) * 16;
    to[i] = c * 1024u;
  }
  const auto copy = [&](int stage, int slot) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      dma::copy16(lds0 + slot * kStage + to[i], woff[i], wrsrc, stage * 2048u);
      dma::copy16(lds0 + slot * kStage + kSide + to[i], xoff[i], xrsrc, stage * 128u);
    }
  };
  const int wc = wave & 1, wr = wave >> 1;  // 128 channels, 64 rows
  // what the results need: a thread's entry of the channels' scales and biases, its rows' scales
  static_assert(kWaves * 64 == 2 * kTile, "a thread to each channel's scale and bias");
  const int channel = b0 * 16 + (threadIdx.x & (kTile - 1));
  const float param = channel < a.n ? (threadIdx.x < kTile ? a.w_scale : a.bias)[(int64_t)e * a.n + channel] : 0.f;
  float xs[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) xs[r] = a.x_scale[min(begin + wr * 64 + r * 32 + (lane & 31), end - 1)];
  v16i acc[4][2];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[c][r][i] = 0;
  const int stages = a.steps / 2;
  copy(0, 0);
  dma::wait_vmcnt<0>();
  __syncthreads();
  // lane's 16 codes of a 32 x 32 block: row lane & 31, codes 16 (lane >> 5) ..
  const uint32_t lane_at = ((lane >> 4) & 1) * 2048u + (lane >> 5) * 256u + (lane & 15) * 16u;
  for (int st = 0; st < stages; ++st) {
    const int slot = st & 1;
    if (st + 1 < stages) copy(st + 1, slot ^ 1);
    const char* wl = lds + slot * kStage + wc * (128 / 16) * 2048 + lane_at;
    const char* xl = lds + slot * kStage + kSide + wr * (64 / 16) * 2048 + lane_at;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int off = (k >> 1) * 1024 + (k & 1) * 512;
      v4i wf[4], xf[2];
#pragma unroll
      for (int c = 0; c < 4; ++c) wf[c] = *reinterpret_cast<const v4i*>(wl + c * 4096 + off);
#pragma unroll
      for (int r = 0; r < 2; ++r) xf[r] = *reinterpret_cast<const v4i*>(xl + r * 4096 + off);
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int r = 0; r < 2; ++r) acc[c][r] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[c], xf[r], acc[c][r], 0, 0, 0);
    }
    dma::wait_vmcnt<0>();
    __syncthreads();
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int r = 0; r < 2; ++r) settle8(acc[c][r]);

  // The results through LDS, 32 rows of a wave's 128 channels at a time, so that
  // whole rows are stored.  A lane has row lane & 31, channels 8 (i / 4) + 4
  // (lane >> 5) + i % 4.
  constexpr int V = kVec<T>, STRIDE = 128 + V;  // the rows that are written together lie in different banks
  T* stage = reinterpret_cast<T*>(lds + 2 * kTile * sizeof(float)) + wave * 32 * STRIDE;
  float* const params = reinterpret_cast<float*>(lds);  // [2][kTile]
  params[threadIdx.x] = param;
  __syncthreads();
  const bool vec = a.n % V == 0 && ((uintptr_t)a.out & 15) == 0;
  const int j0 = b0 * 16 + wc * 128, width = min(128, a.n - j0);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int j = c * 32 + (i >> 2) * 8 + (lane >> 5) * 4;
        const v4f ws = *reinterpret_cast<const v4f*>(params + wc * 128 + j);
        const v4f bias = *reinterpret_cast<const v4f*>(params + kTile + wc * 128 + j);
        float y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) y[u] = finish8<ACT>(acc[c][r][i + u], xs[r] * ws[u], bias[u]);
        Vec<T, 4>::store(stage + (lane & 31) * STRIDE + j, y);
      }
    // the wave's LDS operations are in order; the compiler keeps them so
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int row0 = begin + wr * 64 + r * 32, rows = min(32, end - row0);
    T* out = (T*)a.out + (int64_t)row0 * a.n + j0;
    if (vec) {
      constexpr int PER = 128 / V;  // vectors of a row
      const int c = lane % PER * V;
#pragma unroll
      for (int i = 0; i < 32; i += 64 / PER) {
        const int at = i + lane / PER;
        if (at < rows && c < width)
          *reinterpret_cast<int4*>(out + (int64_t)at * a.n + c) = *reinterpret_cast<const int4*>(stage + at * STRIDE + c);
      }
    } else {
      for (int i = 0; i < rows; ++i)
#pragma unroll
        for (int c = lane; c < 128; c += 64)
          if (c < width) out[(int64_t)i * a.n + c] = stage[i * STRIDE + c];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

template <class T, int ACT>
int tiles_run(const Linear8Args& a, hipStream_t s) {
  constexpr int out = 2 * kTile * (int)sizeof(float) + kWaves * 32 * (128 + kVec<T>) * (int)sizeof(T), bytes = std::max(kLds, out);
  NHIP_TRY(ensure_dynamic_lds((const void*)linear8_tiles_kernel<T, ACT>, bytes));
  const int64_t cols = ceil_div(a.blocks, kTile / 16);
  // every expert's last tile may be a part of one
  const int64_t rows = ceil_div(a.rows, kTile) + (a.starts ? std::min(a.experts, a.rows) : 0);
  if (rows * cols > 0x7fffff00) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "linear8: too many tiles");
  NHIP_LAUNCH("linear8_tiles", (linear8_tiles_kernel<T, ACT>), dim3((uint32_t)round_up(rows * cols, 8)), dim3(kWaves * 64),
              bytes, s, a, (int)cols, (int)(rows * cols));
  return check_launch("linear8_tiles");
}

}  // namespace

bool linear8_tiles_selected(const Linear8Args& a) {
  const int force = setting_int("NHIP_LINEAR8_TILES", -1);
  if (force >= 0) return force != 0;
  return a.rows > 64 * (int64_t)a.experts;
}

int linear8_tiles(const Linear8Args& a, int dtype, hipStream_t s) {
  return NHIP_FOR_ELEM(dtype, T, NHIP_FOR_ACT(a.act, ACT, tiles_run<T, ACT>(a, s)));
}

}  // namespace nhip
