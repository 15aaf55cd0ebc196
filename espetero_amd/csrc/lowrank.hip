// Low-rank adapters of many requests beside a shared projection: Y[row, slice s] += scale[a] * B[a, s] (A[a, s] x[row]) with a the
// row's adapter. The rows of a pass are grouped by adapter into tiles of up to 16 (esp_plan_lowrank); two launches:
//   down  low[split][slot][slices * rank] = x . A^T over the split's share of D, fp32 partial sums in the workspace
//   up    the splits' sums in split order, times B, onto Y
// Every product of two 16-bit elements is exact in fp32 and summed there; the intermediate keeps its 24 bits on its way into the
// second matrix product, which takes 16-bit operands, as the sum of three bf16 or two fp16 numbers.
#include "common.hpp"
#include "lowrank_shape.hpp"

namespace esp {

template <int DT>
__global__ __launch_bounds__(256) void lowrank_down_kernel(const LowRankArgs a) {
  const esp_lowrank_tile tile = a.tiles[blockIdx.x];
  if (tile.count <= 0) return;
  const int split = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, q4 = lane >> 4;
  const int d0 = split * a.chunk, d1 = min(a.D, d0 + a.chunk);
  const int row = a.order[tile.first + min(c16, tile.count - 1)];
  const uint16_t* x = a.X + size_t(row) * a.x_ld;
  const uint16_t* A = a.A + size_t(tile.adapter) * a.n_low * a.D;
  for (int n0 = 16 * wave; n0 < a.n_low; n0 += 64) {
    const uint16_t* ar = A + size_t(min(n0 + c16, a.n_low - 1)) * a.D;
    f32x4 acc = {0, 0, 0, 0};
    for (int d = d0 + 8 * q4; d < d1 + 8 * q4; d += 32) {  // the lanes of a step share its first dim: d1 - d0 steps for all
      const bool in = d < d1;
      const u32x4 xa = in ? *reinterpret_cast<const u32x4*>(ar + d) : u32x4{0, 0, 0, 0};
      const u32x4 xb = in ? *reinterpret_cast<const u32x4*>(x + d) : u32x4{0, 0, 0, 0};
      acc = mfma16x32<DT>(xa, xb, acc);
    }
    mfma_settle(acc);
    if (c16 < tile.count) {
      float* to = a.low + (size_t(split) * a.n_slots + tile.first + c16) * a.n_low + n0 + 4 * q4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n0 + 4 * q4 + e < a.n_low) to[e] = acc[e];
    }
  }
}

// grid: (tiles, blocks of 256 columns of the slices side by side)
template <int DT>
__global__ __launch_bounds__(256) void lowrank_up_kernel(const LowRankArgs a) {
  constexpr int T = DT == ESP_F16 ? 2 : 3;             // 16-bit terms of a number of the intermediate
  __shared__ __attribute__((aligned(16))) uint16_t low[T][16][kLowRankMost + 8];
  __shared__ float unit[16];
  const esp_lowrank_tile tile = a.tiles[blockIdx.x];
  if (tile.count <= 0) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c16 = lane & 15, q4 = lane >> 4;
  int s = 0;                                            // the slice of this block: blocks do not reach over a slice's end
  int blk = blockIdx.y;
  while (s + 1 < a.n_slices && blk >= (a.width[s] + 255) / 256) blk -= (a.width[s++] + 255) / 256;
  int b0 = 0;
  for (int i = 0; i < s; ++i) b0 += a.width[i];
  // The tile's share of the intermediate: splits summed in order, one wavefront per row. An fp16 term holds no more than 65504 and
  // loses bits below 2^-14: a row is taken relative to the power of two at its largest element.
  const int K = (a.rank + 31) / 32 * 32;
  for (int r = wave; r < 16; r += 4) {
    float v[kLowRankMost / 64], most = 0.0f;
#pragma unroll
    for (int i = 0; i < kLowRankMost / 64; ++i) {
      const int k = lane + 64 * i;
      v[i] = 0.0f;
      if (r < tile.count && k < a.rank)
        for (int sp = 0; sp < a.splits; ++sp) v[i] += a.low[(size_t(sp) * a.n_slots + tile.first + r) * a.n_low + s * a.rank + k];
      most = fmaxf(most, fabsf(v[i]));
    }
    float f = 1.0f, back = 1.0f;
    if constexpr (DT == ESP_F16) {
#pragma unroll
      for (int x = 32; x >= 1; x >>= 1) most = fmaxf(most, __shfl_xor(most, x));
      if (most > 0.0f && most < INFINITY) {
        const int e = ilogbf(most);
        f = ldexpf(1.0f, -e);
        back = ldexpf(1.0f, e);
        if (e < -120) f = back = 1.0f;  // so small that its reciprocal's power of two leaves the range
      }
    }
    if (lane == 0) unit[r] = back;
#pragma unroll
    for (int i = 0; i < kLowRankMost / 64; ++i) {
      const int k = lane + 64 * i;
      if (k >= K) continue;
      float rest = v[i] * f;
#pragma unroll
      for (int t = 0; t < T; ++t) {
        const uint16_t w = pack1<DT>(rest);
        low[t][r][k] = w;
        const float had = unpack_lo<DT>(w);
        rest = fabsf(had) < INFINITY ? rest - had : 0.0f;
      }
    }
  }
  __syncthreads();
  const int row = a.order[tile.first + min(c16, tile.count - 1)];
  const float scale = a.scale[tile.adapter] * unit[c16];
  const uint16_t* B = a.B + (size_t(tile.adapter) * a.n_out + b0) * a.rank;
  for (int n0 = 256 * blk + 16 * wave; n0 < min(a.width[s], 256 * blk + 256); n0 += 64) {
    const uint16_t* br = B + size_t(min(n0 + c16, a.width[s] - 1)) * a.rank;
    f32x4 acc = {0, 0, 0, 0};
    for (int k = 0; k < K; k += 32) {
      const u32x4 xa = k + 8 * q4 < a.rank ? *reinterpret_cast<const u32x4*>(br + k + 8 * q4) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int t = 0; t < T; ++t) acc = mfma16x32<DT>(xa, *reinterpret_cast<const u32x4*>(&low[t][c16][k + 8 * q4]), acc);
    }
    mfma_settle(acc);
    if (c16 < tile.count) {
      float* y = a.Y + size_t(row) * a.y_ld + a.y_off[s] + n0 + 4 * q4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n0 + 4 * q4 + e < a.width[s]) y[e] += scale * acc[e];
    }
  }
}

hipError_t launch_lowrank(int dt, const LowRankArgs& a, int n_tiles, hipStream_t st) {
  unsigned blocks = 0;
  for (int s = 0; s < a.n_slices; ++s) blocks += unsigned((a.width[s] + 255) / 256);
  const dim3 down{unsigned(n_tiles), unsigned(a.splits)}, up{unsigned(n_tiles), blocks};
  if (dt == ESP_F16) {
    hipLaunchKernelGGL(lowrank_down_kernel<ESP_F16>, down, dim3(256), 0, st, a);
    hipLaunchKernelGGL(lowrank_up_kernel<ESP_F16>, up, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL(lowrank_down_kernel<ESP_BF16>, down, dim3(256), 0, st, a);
    hipLaunchKernelGGL(lowrank_up_kernel<ESP_BF16>, up, dim3(256), 0, st, a);
  }
  return hipGetLastError();
}

}  // namespace esp
