// Low-rank adapters of many requests beside a shared projection: Y[row, slice s] += scale[a] * B[a, s] (A[a, s] x[row]) with a the
// row's adapter. The rows of a pass are grouped by adapter into tiles of up to 16 or 64 (esp_plan_lowrank); two launches:
//   down  low[split][slot][slices * rank] = x . A^T over the split's share of D, fp32 partial sums in the workspace
//   up    the splits' sums in split order, times B, onto Y
// Every product of two 16-bit elements is exact in fp32 and summed there; the intermediate keeps its 24 bits on its way into the
// second matrix product, which takes 16-bit operands, as the sum of three bf16 or two fp16 numbers.
#include "common.hpp"
#include "lowrank_shape.hpp"

namespace esp {

// An fp16 term holds no more than 65504 and loses bits below 2^-14: a row of the intermediate is taken relative to the power of two
// at its largest element, whose bits these are. 0 for a row of zeros or infinities, or one whose reciprocal leaves the range.
__device__ __forceinline__ int power_of(uint32_t most) {
  const int e = int(most >> 23) - 127;
  return e < -120 || e > 127 ? 0 : min(e, 126);
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }

// Four numbers as T terms of 16 bits, `apart` elements from one term to the next.
template <int DT, int T>
__device__ __forceinline__ void put_terms(f32x4 rest, uint16_t* to, int apart) {
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const u32x2 w = {pack2<DT>(rest[0], rest[1]), pack2<DT>(rest[2], rest[3])};
    *reinterpret_cast<u32x2*>(to + t * apart) = w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float had = e & 1 ? unpack_hi<DT>(w[e >> 1]) : unpack_lo<DT>(w[e >> 1]);
      rest[e] = fabsf(had) < INFINITY ? rest[e] - had : 0.0f;
    }
  }
}

// Columns c .. c + 3 of a row of Y, of which those before the slice's end are there; `was`: what all four held.
__device__ __forceinline__ void add_to(float* y, int c, int width, f32x4 was, float f, f32x4 sum) {
  if (c + 4 <= width) {
    const f32x4 now = was + f * sum;
    __builtin_memcpy(y + c, &now, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < width) y[c + e] += f * sum[e];
  }
}

// grid: (splits, tiles, groups of 16 NB rows of A): with eight splits each XCD has its own share of the dims, so no two L2s hold the
// same elements. Of its workgroup's share of the dims a wavefront takes 32 at a time, each with
// all of the tile's 16 R rows and the group's rows of A, so no element is read by two of them; their sums meet in LDS.
template <int DT, int R, int NB>
__global__ __launch_bounds__(256) void lowrank_down_kernel(const LowRankArgs a) {
  constexpr int F = R * NB, AHEAD = R == 1 ? 6 : 4;
  __shared__ f32x4 part[2][F][64];
  const esp_lowrank_tile tile = a.tiles[blockIdx.y];
  if (tile.count <= 0) return;
  const int split = blockIdx.x, n0 = blockIdx.z * 16 * NB, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, q4 = lane >> 4;
  const uint16_t *x[R], *ar[NB];
#pragma unroll
  for (int r = 0; r < R; ++r) x[r] = a.X + size_t(a.order[tile.first + min(16 * r + c16, tile.count - 1)]) * a.x_ld + 8 * q4;
#pragma unroll
  for (int b = 0; b < NB; ++b) ar[b] = a.A + (size_t(tile.adapter) * a.n_low + min(n0 + 16 * b + c16, a.n_low - 1)) * a.D + 8 * q4;
  struct Step {
    u32x4 x[R], a[NB];
  } ring[AHEAD];
  auto load = [&](Step& s, int d) {
#pragma unroll
    for (int r = 0; r < R; ++r) s.x[r] = *reinterpret_cast<const u32x4*>(x[r] + d);
#pragma unroll
    for (int b = 0; b < NB; ++b) s.a[b] = *reinterpret_cast<const u32x4*>(ar[b] + d);
  };
  f32x4 acc[R][NB];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[r][b] = f32x4{0, 0, 0, 0};
  const int d0 = split * a.chunk, d1 = min(a.D, d0 + a.chunk);
  const int whole = a.D / 32 * 32, steps = (max(0, min(whole, d1) - d0 - 32 * wave) + 127) / 128;
  auto dim = [&](int s) { return d0 + 32 * (wave + 4 * s); };
  for (int s0 = 0; s0 < steps; s0 += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s0 + i < steps) load(ring[i], dim(s0 + i));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (s0 + i < steps) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r][b] = mfma16x32<DT>(ring[i].a[b], ring[i].x[r], acc[r][b]);
      }
    }
  }
  if (whole < a.D && wave == 0 && d0 <= whole && whole < d1) {  // the dims behind the last 32: lanes behind D add zeros
    const bool in = whole + 8 * q4 < a.D;
    u32x4 tx[R];
#pragma unroll
    for (int r = 0; r < R; ++r) tx[r] = in ? *reinterpret_cast<const u32x4*>(x[r] + whole) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const u32x4 ta = in ? *reinterpret_cast<const u32x4*>(ar[b] + whole) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r][b] = mfma16x32<DT>(ta, tx[r], acc[r][b]);
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      mfma_settle(acc[r][b]);
      if (wave >= 2) part[wave - 2][r * NB + b][lane] = acc[r][b];
    }
  __syncthreads();
  if (wave < 2) {
#pragma unroll
    for (int f = 0; f < F; ++f) part[wave][f][lane] += acc[f / NB][f % NB];
  }
  __syncthreads();
  for (int f = wave; f < F; f += 4) {
    const f32x4 s = part[0][f][lane] + part[1][f][lane];
    const int row = 16 * (f / NB) + c16, n = n0 + 16 * (f % NB) + 4 * q4;
    if (row < tile.count && n < a.n_low) *reinterpret_cast<f32x4*>(a.low + (size_t(split) * a.n_slots + tile.first + row) * a.n_low + n) = s;
  }
}

// grid: eight tiles after each other, then the next block of 256 columns of the slices side by side for them: a tile's blocks are on
// one XCD, whose L2 then serves all but the first with the tile's intermediate. A wavefront takes 64 columns with all of the tile's rows. What it
// reads of Y and B is on its way while the splits are summed.
template <int DT, int R, int MOST>
__global__ __launch_bounds__(256, 2) void lowrank_up_kernel(const LowRankArgs a, int n_tiles, int blocks) {
  constexpr int T = DT == ESP_F16 ? 2 : 3;  // 16-bit terms of a number of the intermediate
  constexpr int Q = R * 16 * (MOST / 4) / 256, SB = R == 1 ? 8 : 4;  // loads of a thread from a split, splits on their way at once
  extern __shared__ __attribute__((aligned(16))) uint16_t low[];  // [T][16 R][K + 8]
  __shared__ uint32_t most[16 * R];
  const int of_xcd = blockIdx.x >> 3, eight = of_xcd / blocks, which = 8 * eight + (blockIdx.x & 7);
  if (which >= n_tiles) return;
  const esp_lowrank_tile tile = a.tiles[which];
  if (tile.count <= 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, q4 = lane >> 4;
  int s = 0, b0 = 0, blk = of_xcd - eight * blocks;  // the slice of this block: blocks do not reach over a slice's end
  while (s + 1 < a.n_slices && blk >= (a.width[s] + 255) / 256) blk -= (a.width[s] + 255) / 256, b0 += a.width[s++];
  const float scale = a.scale[tile.adapter];
  const int K = (a.rank + 31) / 32 * 32, ld = K + 8, width = a.width[s], c0 = 256 * blk + 64 * wave;
  float* y[R];
#pragma unroll
  for (int r = 0; r < R; ++r) y[r] = a.Y + size_t(a.order[tile.first + min(16 * r + c16, tile.count - 1)]) * a.y_ld + a.y_off[s];
  const uint16_t* B = a.B + (size_t(tile.adapter) * a.n_out + b0) * a.rank;
  // The splits' sums: a thread has four numbers of a row at a time.
  const int splits = a.splits, n_low = a.n_low;
  const size_t per_split = size_t(a.n_slots) * n_low;
  const float* const low_sums = a.low + size_t(tile.first) * n_low + s * a.rank;
  const int quads = a.rank / 4, per = 65536 / quads + 1;
  auto row_of = [&](int at) { return at * per >> 16; };  // at / quads, for at < 2048 and quads <= 32
  f32x4 v[Q], some[SB][Q];
  uint32_t from[Q];  // bytes; rows behind the tile's see its last again
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = tid + 256 * i, row = row_of(at);
    from[i] = uint32_t(min(row, tile.count - 1) * n_low + (at - row * quads) * 4) * 4;
    v[i] = f32x4{0, 0, 0, 0};
  }
  auto load_low = [&](int sp0) {
#pragma unroll
    for (int sp = 0; sp < SB; ++sp) {
      const char* const base = reinterpret_cast<const char*>(low_sums + min(sp0 + sp, splits - 1) * per_split);
#pragma unroll
      for (int i = 0; i < Q; ++i) some[sp][i] = *reinterpret_cast<const f32x4*>(base + from[i]);
    }
  };
  auto add_low = [&](int sp0) {
#pragma unroll
    for (int sp = 0; sp < SB; ++sp)
      if (sp0 + sp < splits) {
#pragma unroll
        for (int i = 0; i < Q; ++i) v[i] += some[sp][i];
      }
  };
  int sp0 = 0;
  for (; sp0 + SB < splits; sp0 += SB) {
    load_low(sp0);
    __builtin_amdgcn_sched_barrier(0);
    add_low(sp0);
  }
  load_low(sp0);
  // Y, and the first 32 of every column's rank. Columns behind the slice's end see its last ones again.
  f32x4 was[R][4];
  u32x4 bq[4];
  const bool wide = width >= 4;
  auto load_b = [&](int k) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint16_t* from = B + size_t(min(c0 + 16 * n + c16, width - 1)) * a.rank;
      bq[n] = *reinterpret_cast<const u32x4*>(from + (k + 8 * q4 < a.rank ? k + 8 * q4 : 0));
    }
  };
  if (wide) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < 4; ++n) __builtin_memcpy(&was[r][n], y[r] + min(c0 + 16 * n + 4 * q4, width - 4), 16);
  }
  load_b(0);
  __builtin_amdgcn_sched_barrier(0);
  add_low(sp0);
  // An fp16 term holds no more than 65504 and loses bits below 2^-14: a row is taken relative to the power of two at its largest.
  if constexpr (DT == ESP_F16) {
    if (tid < 16 * R) most[tid] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int row = row_of(tid + 256 * i);
      if (row < tile.count) atomicMax(&most[row], __float_as_uint(fmaxf(fmaxf(fabsf(v[i][0]), fabsf(v[i][1])), fmaxf(fabsf(v[i][2]), fabsf(v[i][3])))));
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = tid + 256 * i, row = row_of(at), k = (at - row * quads) * 4;
    if (row >= 16 * R) continue;
    const float f = DT == ESP_F16 ? two_to(-power_of(most[row])) : 1.0f;
    put_terms<DT, T>(v[i] * f, &low[row * ld + k], 16 * R * ld);
  }
  for (int at = tid; at < T * 16 * R * (K - a.rank) / 4; at += 256) {  // the zeros up to K
    const int gap = (K - a.rank) / 4;
    *reinterpret_cast<u32x2*>(&low[at / gap * ld + a.rank + at % gap * 4]) = u32x2{0, 0};
  }
  __syncthreads();
  if (c0 >= width) return;
  f32x4 acc[R][4];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[r][n] = f32x4{0, 0, 0, 0};
  for (int k = 0; k < K; k += 32) {
    if (k) load_b(k);
    if (k + 8 * q4 >= a.rank) bq[0] = bq[1] = bq[2] = bq[3] = u32x4{0, 0, 0, 0};  // lanes behind the rank
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const u32x4 l = *reinterpret_cast<const u32x4*>(&low[((t * R + r) * 16 + c16) * ld + k + 8 * q4]);
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[r][n] = mfma16x32<DT>(bq[n], l, acc[r][n]);
      }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int row = 16 * r + c16;
    float f = scale;
    if constexpr (DT == ESP_F16) f *= two_to(power_of(most[row]));
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      mfma_settle(acc[r][n]);
      const int c = c0 + 16 * n + 4 * q4;
      if (row < tile.count) add_to(y[r], c, width, was[r][n], f, acc[r][n]);
    }
  }
}

// Both products in one launch, for tiles of 16 rows and little of A: grid (tiles, blocks of 1024 columns). Every workgroup sums its
// slice's intermediate for itself, each of the 16 wavefronts over its own dims, and adds 64 columns a wavefront to Y.
template <int DT, int NB>
__global__ __launch_bounds__(1024) void lowrank_fused_kernel(const LowRankArgs a) {
  constexpr int T = DT == ESP_F16 ? 2 : 3, K = NB == 1 ? 32 : 16 * NB, AHEAD = NB == 1 ? 4 : 2;
  __shared__ f32x4 part[16][NB][64];
  __shared__ __attribute__((aligned(16))) uint16_t low[T][16][K + 8];
  __shared__ uint32_t most[16];
  const esp_lowrank_tile tile = a.tiles[blockIdx.x];
  if (tile.count <= 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c16 = lane & 15, q4 = lane >> 4;
  int s = 0, b0 = 0, blk = blockIdx.y;
  while (s + 1 < a.n_slices && blk >= (a.width[s] + 1023) / 1024) blk -= (a.width[s] + 1023) / 1024, b0 += a.width[s++];
  const int width = a.width[s], c0 = 1024 * blk + 64 * wave;
  const bool mine = c16 < tile.count;
  const float scale = a.scale[tile.adapter];
  const int row = a.order[tile.first + min(c16, tile.count - 1)];
  const uint16_t* const x = a.X + size_t(row) * a.x_ld + 8 * q4;
  const uint16_t* ar[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) ar[b] = a.A + (size_t(tile.adapter) * a.n_low + s * a.rank + min(16 * b + c16, a.rank - 1)) * a.D + 8 * q4;
  float* const y = a.Y + size_t(row) * a.y_ld + a.y_off[s];
  const uint16_t* const B = a.B + (size_t(tile.adapter) * a.n_out + b0) * a.rank;
  u32x4 xr[AHEAD], av[AHEAD][NB];
  const int steps = (max(0, a.D / 32 - wave) + 15) / 16;
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (s0 + i < steps) {
        const int d = 32 * (wave + 16 * (s0 + i));
#pragma unroll
        for (int b = 0; b < NB; ++b) av[i][b] = *reinterpret_cast<const u32x4*>(ar[b] + d);
        xr[i] = *reinterpret_cast<const u32x4*>(x + d);
      }
  };
  f32x4 acc[NB], was[4];
  u32x4 bq[K / 32][4];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x4{0, 0, 0, 0};
  load(0);
  // What the second product needs comes behind them. Columns behind the slice's end see its last ones again.
  const bool wide = width >= 4 && c0 < width;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if (wide) __builtin_memcpy(&was[n], y + min(c0 + 16 * n + 4 * q4, width - 4), 16);
    if (c0 >= width) continue;
    const uint16_t* from = B + size_t(min(c0 + 16 * n + c16, width - 1)) * a.rank;
#pragma unroll
    for (int k = 0; k < K / 32; ++k) {
      bq[k][n] = *reinterpret_cast<const u32x4*>(from + (32 * k + 8 * q4 < a.rank ? 32 * k + 8 * q4 : 0));
    }
  }
  if (tid < 16) most[tid] = 0;
  for (int s0 = 0; s0 < steps; s0 += AHEAD) {
    if (s0) load(s0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (s0 + i < steps) {
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = mfma16x32<DT>(av[i][b], xr[i], acc[b]);
      }
    }
  }
  if (a.D % 32 && wave == 15) {
    const int d = a.D / 32 * 32;
    const bool in = d + 8 * q4 < a.D;
    const u32x4 tx = in ? *reinterpret_cast<const u32x4*>(x + d) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = mfma16x32<DT>(in ? *reinterpret_cast<const u32x4*>(ar[b] + d) : u32x4{0, 0, 0, 0}, tx, acc[b]);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    mfma_settle(acc[b]);
    part[wave][b][lane] = acc[b];
  }
  __syncthreads();
  // Wavefront b joins the sums of 16 rows of A, and those that only fill up K are zeros.
  f32x4 v = {0, 0, 0, 0};
  if (wave < NB) {
#pragma unroll
    for (int w = 0; w < 16; ++w) v += part[w][wave < NB ? wave : 0][lane];
    if (16 * wave + 4 * q4 >= a.rank) v = f32x4{0, 0, 0, 0};
  }
  int e = 0;
  if constexpr (DT == ESP_F16) {
    if (wave < NB) atomicMax(&most[c16], __float_as_uint(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])))));
    __syncthreads();
    e = power_of(most[c16]);
  }
  if (wave < K / 16) put_terms<DT, T>(v * two_to(-e), &low[0][c16][16 * wave + 4 * q4], 16 * (K + 8));
  __syncthreads();
  if (c0 >= width) return;
  if (K - 32 + 8 * q4 >= a.rank) {  // lanes behind the rank
#pragma unroll
    for (int n = 0; n < 4; ++n) bq[K / 32 - 1][n] = u32x4{0, 0, 0, 0};
  }
  const float f = scale * two_to(e);
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < K / 32; ++k)
#pragma unroll
      for (int t = 0; t < T; ++t) sum = mfma16x32<DT>(bq[k][n], *reinterpret_cast<const u32x4*>(&low[t][c16][32 * k + 8 * q4]), sum);
    mfma_settle(sum);
    if (mine) add_to(y, c0 + 16 * n + 4 * q4, width, was[n], f, sum);
  }
}

template <int DT, int NB>
static void run_fused(const LowRankArgs& a, int n_tiles, hipStream_t st) {
  unsigned blocks = 0;
  for (int s = 0; s < a.n_slices; ++s) blocks += unsigned((a.width[s] + 1023) / 1024);
  hipLaunchKernelGGL((lowrank_fused_kernel<DT, NB>), dim3(unsigned(n_tiles), blocks), dim3(1024), 0, st, a);
}

template <int DT, int R>
static hipError_t run_lowrank(const LowRankArgs& a, int n_tiles, hipStream_t st) {
  const int nb = lowrank_low_blocks(a.n_low);
  const dim3 down{unsigned(a.splits), unsigned(n_tiles), unsigned(lowrank_low_groups(a.n_low))};
  if (nb == 1) hipLaunchKernelGGL((lowrank_down_kernel<DT, R, 1>), down, dim3(256), 0, st, a);
  else if (nb == 2) hipLaunchKernelGGL((lowrank_down_kernel<DT, R, 2>), down, dim3(256), 0, st, a);
  else if (nb == 3) hipLaunchKernelGGL((lowrank_down_kernel<DT, R, 3>), down, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((lowrank_down_kernel<DT, R, 4>), down, dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  unsigned blocks = 0;
  for (int s = 0; s < a.n_slices; ++s) blocks += unsigned((a.width[s] + 255) / 256);
  const dim3 up{unsigned(n_tiles + 7) / 8 * 8 * blocks};
  const size_t lds = size_t(DT == ESP_F16 ? 2 : 3) * 16 * R * ((a.rank + 31) / 32 * 32 + 8) * 2;
  if (R == 4 && a.rank <= 16) hipLaunchKernelGGL((lowrank_up_kernel<DT, 4, 16>), up, dim3(256), lds, st, a, n_tiles, int(blocks));
  else if (R == 4 && a.rank <= 32) hipLaunchKernelGGL((lowrank_up_kernel<DT, 4, 32>), up, dim3(256), lds, st, a, n_tiles, int(blocks));
  else if (a.rank <= 64) hipLaunchKernelGGL((lowrank_up_kernel<DT, R, 64>), up, dim3(256), lds, st, a, n_tiles, int(blocks));
  else hipLaunchKernelGGL((lowrank_up_kernel<DT, R, 128>), up, dim3(256), lds, st, a, n_tiles, int(blocks));
  return hipGetLastError();
}

template <int DT>
static hipError_t run_any(const LowRankArgs& a, int rows_per_tile, int n_tiles, hipStream_t st) {
  if (rows_per_tile != 16) return run_lowrank<DT, 4>(a, n_tiles, st);
  if (!lowrank_fused(a.D, a.rank, a.n_slices, a.width, n_tiles)) return run_lowrank<DT, 1>(a, n_tiles, st);
  if (a.rank <= 16) run_fused<DT, 1>(a, n_tiles, st);
  else if (a.rank <= 32) run_fused<DT, 2>(a, n_tiles, st);
  else run_fused<DT, 4>(a, n_tiles, st);
  return hipGetLastError();
}

hipError_t launch_lowrank(int dt, const LowRankArgs& a, int rows_per_tile, int n_tiles, hipStream_t st) {
  return dt == ESP_F16 ? run_any<ESP_F16>(a, rows_per_tile, n_tiles, st) : run_any<ESP_BF16>(a, rows_per_tile, n_tiles, st);
}

}  // namespace esp
