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

template <class T>
__global__ __launch_bounds__(kWaves * 64) void linear8_tiles_kernel(Linear8Args a, int col_tiles, int work) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups go to the eight dies in turn: each die gets a run of the tiles
  const int id = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
  if (id >= work) return;
  int e, begin, end;
  if (!find_tile(a, id / col_tiles, e, begin, end)) return;
  const int b0 = id % col_tiles * (kTile / 16);  // first block of channels
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

  // lane: row lane & 31 of the 32, channels 8 (i / 4) + 4 (lane >> 5) + i % 4
  const float* ws = a.w_scale + (int64_t)e * a.n;
  const float* bias = a.bias + (int64_t)e * a.n;
  const bool vec = a.n % 4 == 0 && ((uintptr_t)a.out & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = begin + wr * 64 + r * 32 + (lane & 31);
    if (row >= end) continue;
    const float xs = a.x_scale[row];
    T* out = (T*)a.out + (int64_t)row * a.n;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int j = b0 * 16 + wc * 128 + c * 32 + (i >> 2) * 8 + (lane >> 5) * 4;
        float y[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          y[u] = finish8(acc[c][r][i + u], xs * ws[min(j + u, a.n - 1)], bias[min(j + u, a.n - 1)], a.act);
        if (vec && j < a.n)
          Vec<T, 4>::store(out + j, y);
        else
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (j + u < a.n) out[j + u] = (T)y[u];
      }
  }
}

template <class T>
int tiles_run(const Linear8Args& a, hipStream_t s) {
  NHIP_TRY(ensure_dynamic_lds((const void*)linear8_tiles_kernel<T>, kLds));
  const int64_t cols = ceil_div(a.blocks, kTile / 16);
  // every expert's last tile may be a part of one
  const int64_t rows = ceil_div(a.rows, kTile) + (a.starts ? std::min(a.experts, a.rows) : 0);
  if (rows * cols > 0x7fffff00) return fail(NHIP_STATUS_SHAPE_ARITHMETIC_OVERFLOW, "linear8: too many tiles");
  NHIP_LAUNCH("linear8_tiles", linear8_tiles_kernel<T>, dim3((uint32_t)round_up(rows * cols, 8)), dim3(kWaves * 64), kLds, s, a,
              (int)cols, (int)(rows * cols));
  return check_launch("linear8_tiles");
}

}  // namespace

bool linear8_tiles_selected(const Linear8Args& a) {
  const int force = setting_int("NHIP_LINEAR8_TILES", -1);
  if (force >= 0) return force != 0;
  return a.rows > 64 * (int64_t)a.experts;
}

int linear8_tiles(const Linear8Args& a, int dtype, hipStream_t s) {
  return NHIP_FOR_ELEM(dtype, T, tiles_run<T>(a, s));
}

}  // namespace nhip
