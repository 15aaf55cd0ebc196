// Low-rank adapters of many requests beside a shared projection: Y[row, slice s] += scale[a] * B[a, s] (A[a, s] x[row]) with a the
// row's adapter. The rows of a pass are grouped by adapter into tiles of up to 16 or 64 (esp_plan_lowrank); two launches:
//   down  low[split][slot][slices * rank] = x . A^T over the split's share of D, fp32 partial sums in the workspace
//   up    the splits' sums in split order, times B, onto Y
// or one that does both where there is little of A. Prompts are bound by Y, read and written once: 3679 rows of 7168 columns, rank 16,
// D 5120 take 51 us, 4.9 TB/s. A decode batch is bound by the hops from record to row number to element, about a microsecond each, and by
// the second launch: 48 requests of 20 adapters, rank 16, D 5120 take 11 us (4 + 6 in the kernels), of which its 16 MB are 3.
// Every product of two 16-bit elements is exact in fp32 and summed there. On its way into the second matrix product, which takes 16-bit
// operands, an intermediate becomes the sum of three bf16 numbers, which keep its 24 bits, or of two fp16 ones. Those keep it to 2^-23
// of itself, or to 2^-39 of the row's largest where that is more (a number of 2^-16 of the largest or less). A third would keep the
// last bit too and cost half as many products again.
#include "common.hpp"
#include "lowrank_shape.hpp"

#include <type_traits>

namespace esp {

// An fp16 term holds no more than 65504 and loses bits below 2^-14: a row of the intermediate is taken relative to a power of two that
// puts its largest element, whose bits these are, at 2^14 .. 2^15, as far from the loss as there is room. (Rows of zeros and infinities
// stay what they are; two_to has the power and its reciprocal.)
__device__ __forceinline__ int power_of(uint32_t most) { return max(-112, min(int(most >> 23) - 127, 127)) - 14; }
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

// grid: (splits, tiles, groups of 16 NB rows of A): with eight splits each XCD has its own share of the dims, so no two L2s hold the
// same elements. 128 dims at a time of the tile's 16 R rows and the group's rows of A go through LDS, two turns ahead in registers.
// They cannot come from memory as the matrix product takes them, 16 lanes on 16 rows: a load then looks up 64 lines instead of 8,
// and the prompts' launch, bound by that, took 17 us instead of 11. Of tiles of 64 rows a wavefront has 16; of tiles of 16 every
// fourth 32 dims, and their sums meet in LDS.
template <int DT, int R, int NB>
__global__ __launch_bounds__(256) void lowrank_down_kernel(const LowRankArgs a) {
  constexpr int L = R + NB, KS = R == 1 ? 1 : 4;  // loads of a thread a turn, and 32s of dims of a wavefront in it
  static_assert(R == 1 || R == 4);
  __shared__ u32x4 stage[16 * L][16];             // 16 bytes c of row r at c ^ r % 16
  const esp_lowrank_tile tile = a.tiles[blockIdx.y];
  if (tile.count <= 0) return;
  const int split = blockIdx.x, n0 = blockIdx.z * 16 * NB, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, q4 = lane >> 4, part = tid & 15, mine = tid >> 4;  // the thread's 16 bytes, and its row of every 16
  const uint16_t* from[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    if (i < R) from[i] = a.X + size_t(a.order[tile.first + min(16 * i + mine, tile.count - 1)]) * a.x_ld;
    else from[i] = a.A + (size_t(tile.adapter) * a.n_low + min(n0 + 16 * (i - R) + mine, a.n_low - 1)) * a.D;
  }
  const int D = a.D, d0 = split * a.chunk, d1 = min(D, d0 + a.chunk);
  auto load = [&](u32x4 (&to)[L], int d) {  // dims behind D: the row's first, and no part of the sums
    const int at = d + 8 * part < D ? d + 8 * part : 0;
#pragma unroll
    for (int i = 0; i < L; ++i) to[i] = *reinterpret_cast<const u32x4*>(from[i] + at);
  };
  f32x4 acc[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x4{0, 0, 0, 0};
  auto turn = [&](u32x4 (&held)[L], int d) {
    const bool in = d + 8 * part < D;
#pragma unroll
    for (int i = 0; i < L; ++i) stage[16 * i + mine][part ^ mine] = in ? held[i] : u32x4{0, 0, 0, 0};
    __syncthreads();
    if (d + 256 < d1) load(held, d + 256);
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const int c = (4 * (R == 1 ? wave : k) + q4) ^ c16;
      const u32x4 x = stage[(R == 1 ? 0 : 16 * wave) + c16][c];
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = mfma16x32<DT>(x, stage[16 * (R + b) + c16][c], acc[b]);
    }
    __syncthreads();
  };
  u32x4 even[L], odd[L];
  if (d0 < d1) load(even, d0);
  if (d0 + 128 < d1) load(odd, d0 + 128);
  for (int d = d0; d < d1; d += 256) {
    turn(even, d);
    if (d + 128 < d1) turn(odd, d + 128);
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) mfma_settle(acc[b]);
  float* const to = a.low + (size_t(split) * a.n_slots + tile.first) * a.n_low + n0 + c16;  // a lane: four rows of one column
  if constexpr (R == 1) {
    f32x4 (*sums)[64] = reinterpret_cast<f32x4 (*)[64]>(stage);                             // [wavefront, block of columns][lane]
#pragma unroll
    for (int b = 0; b < NB; ++b) sums[wave * NB + b][lane] = acc[b];
    __syncthreads();
    if (wave >= NB) return;
    const f32x4 s = (sums[wave][lane] + sums[NB + wave][lane]) + (sums[2 * NB + wave][lane] + sums[3 * NB + wave][lane]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (4 * q4 + e < tile.count && n0 + 16 * wave + c16 < a.n_low) to[size_t(4 * q4 + e) * a.n_low + 16 * wave] = s[e];
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 16 * wave + 4 * q4 + e;
        if (row < tile.count && n0 + 16 * b + c16 < a.n_low) to[size_t(row) * a.n_low + 16 * b] = acc[b][e];
      }
  }
}

// grid: eight tiles after each other, then the next block of 256 columns of the slices side by side for them: a tile's blocks are on
// one XCD, whose L2 then serves all but the first with the tile's intermediate. A wavefront takes 64 columns (32 of tiles of 64 rows)
// with all of the tile's rows. What it reads of Y and B is on its way while the splits are summed; B goes through LDS, 64 of the rank
// at a time, for the same reason as above. A lane has columns 2 i and 2 i + 1 of a 32, so 16 lanes read and write a whole line of Y.
template <int DT, int R, int MOST>
__global__ __launch_bounds__(256, R == 1 ? 4 : 3) void lowrank_up_kernel(const LowRankArgs a, int n_tiles, int blocks, int each) {
  constexpr int T = DT == ESP_F16 ? 2 : 3;  // 16-bit terms of a number of the intermediate
  constexpr int W = 256, CN = R == 1 ? 2 : 1, CB = 128 * CN;  // threads, 32s of columns of a wavefront, columns of the workgroup
  constexpr int Q = (R * 16 * (MOST / 4) + W - 1) / W, SB = Q > 4 ? 2 : R == 4 || Q > 1 ? 4 : 8;  // loads of a thread from a split, splits on their way at once
  constexpr int BQ = CB * 8 / W, BL = 64 + 8;         // 16 bytes of B of a thread at a time, elements of a column in LDS
  extern __shared__ __attribute__((aligned(16))) uint16_t low[];  // [T][16 R][K + 8]
  __shared__ __attribute__((aligned(16))) uint16_t b_sh[R == 1 ? 8 : CB * BL];
  __shared__ uint32_t most[16 * R];
  __shared__ int32_t rows_sh[16 * R];
  const int of_xcd = blockIdx.x >> 3, eight = of_xcd / blocks, which = 8 * eight + (blockIdx.x & 7);
  if (which >= n_tiles) return;
  const esp_lowrank_tile tile = a.tiles[which];
  if (tile.count <= 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c16 = lane & 15, q4 = lane >> 4;
  int s = 0, b0 = 0, blk = of_xcd - eight * blocks;  // the slice of these blocks: they do not reach over a slice's end
  auto runs = [&](int s) { return (a.width[s] + CB * each - 1) / (CB * each); };
  while (s + 1 < a.n_slices && blk >= runs(s)) blk -= runs(s), b0 += a.width[s++];
  const float scale = a.scale[tile.adapter];
  const int rank = a.rank, K = (rank + 31) / 32 * 32, ld = K + 8, width = a.width[s], w0 = 32 * CN * wave;
  int first = CB * each * blk;
  const int last = min(width, first + CB * each);
  if (tid < 16 * R) {  // rows behind the tile's see its last again
    rows_sh[tid] = a.order[tile.first + min(tid, tile.count - 1)];
    most[tid] = 0;
  }
  // The splits' sums: a thread has four numbers of a row at a time.
  const int splits = a.splits, n_low = a.n_low;
  const size_t per_split = size_t(a.n_slots) * n_low;
  const float* const low_sums = a.low + size_t(tile.first) * n_low + s * rank;
  const int quads = rank / 4, per = 65536 / quads + 1;
  auto row_of = [&](int at) { return at * per >> 16; };  // at / quads, for at < 2048 and quads <= 32
  f32x4 v[Q], some[SB][Q];
  uint32_t from[Q];  // bytes
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = tid + W * i, row = row_of(at);
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
  // The block's columns of B, 64 of the rank, and what lies behind the rank or the slice as zeros. Few rows take them from memory as
  // they go into the products: that is one barrier less, and there is little of it.
  constexpr bool LDS = R > 1;
  u32x4 b_held[BQ];
  auto load_b = [&](int k0) {
#pragma unroll
    for (int i = 0; i < BQ; ++i) {
      const int at = tid + W * i, c = LDS ? at / 8 : w0 + 32 * (i / 4) + 2 * c16 + (i / 2 & 1), k = k0 + (LDS ? at % 8 * 8 : 32 * (i & 1) + 8 * q4);
      b_held[i] = *reinterpret_cast<const u32x4*>(a.B + (size_t(tile.adapter) * a.n_out + b0 + min(first + c, width - 1)) * rank + (k < rank ? k : 0));
    }
  };
  auto put_b = [&](int k0) {
#pragma unroll
    for (int i = 0; i < BQ; ++i) {
      const int at = tid + W * i, k = k0 + (LDS ? at % 8 * 8 : 32 * (i & 1) + 8 * q4);
      b_held[i] = k < rank ? b_held[i] : u32x4{0, 0, 0, 0};
      if constexpr (LDS) *reinterpret_cast<u32x4*>(&b_sh[at / 8 * BL + at % 8 * 8]) = b_held[i];
    }
  };
  load_b(0);
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (R > 1) add_low(sp0);  // Y's registers are the splits' until here
  __syncthreads();
  // Y; columns behind the slice's end see its last again.
  float2 was[R][4][CN];
  float* const Y = a.Y + a.y_off[s];
  const int y_ld = a.y_ld;
  auto load_y = [&] {
    if (width < 2) return;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float* const y = Y + int64_t(rows_sh[16 * r + 4 * q4 + e]) * y_ld;
#pragma unroll
        for (int n = 0; n < CN; ++n) __builtin_memcpy(&was[r][e][n], y + max(0, min(first + w0 + 32 * n + 2 * c16, width - 2)), 8);
      }
  };
  load_y();
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (R == 1) add_low(sp0);
  if constexpr (DT == ESP_F16) {
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int row = row_of(tid + W * i);
      if (row < tile.count) atomicMax(&most[row], __float_as_uint(fmaxf(fmaxf(fabsf(v[i][0]), fabsf(v[i][1])), fmaxf(fabsf(v[i][2]), fabsf(v[i][3])))));
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const int at = tid + W * i, row = row_of(at), k = (at - row * quads) * 4;
    if (row >= 16 * R) continue;
    const float f = DT == ESP_F16 ? two_to(-power_of(most[row])) : 1.0f;
    put_terms<DT, T>(v[i] * f, &low[row * ld + k], 16 * R * ld);
  }
  for (int at = tid; at < T * 16 * R * (K - rank) / 4; at += W) {  // the zeros up to K
    const int gap = (K - rank) / 4;
    *reinterpret_cast<u32x2*>(&low[at / gap * ld + rank + at % gap * 4]) = u32x2{0, 0};
  }
  for (;;) {
    f32x4 acc[R][CN][2];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < CN; ++n) acc[r][n][0] = acc[r][n][1] = f32x4{0, 0, 0, 0};
    for (int k0 = 0; k0 < K; k0 += 64) {
      if (LDS && k0) __syncthreads();
      if (!LDS && k0) load_b(k0);
      put_b(k0);
      if (LDS || !k0) __syncthreads();
      if (LDS && k0 + 64 < K) load_b(k0 + 64);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = k0 + 32 * h;
        if (k >= K) break;
        u32x4 bq[CN][2];
#pragma unroll
        for (int n = 0; n < CN; ++n)
#pragma unroll
          for (int o = 0; o < 2; ++o) bq[n][o] = !LDS ? b_held[(4 * n + 2 * o + h) % BQ] : *reinterpret_cast<const u32x4*>(&b_sh[(w0 + 32 * n + 2 * c16 + o) * BL + 32 * h + 8 * q4]);
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const u32x4 l = *reinterpret_cast<const u32x4*>(&low[((t * R + r) * 16 + c16) * ld + k + 8 * q4]);
#pragma unroll
            for (int n = 0; n < CN; ++n)
#pragma unroll
              for (int o = 0; o < 2; ++o) acc[r][n][o] = mfma16x32<DT>(l, bq[n][o], acc[r][n][o]);
            if (R > 1 && r % 2) __builtin_amdgcn_sched_barrier(0);  // no more operands on their way than there are registers for
          }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int n = 0; n < CN; ++n) mfma_settle(acc[r][n][0]), mfma_settle(acc[r][n][1]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 16 * r + 4 * q4 + e;
        if (row >= tile.count) continue;
        float f = scale;
        if constexpr (DT == ESP_F16) f *= two_to(power_of(most[row]));
        float* const y = Y + int64_t(rows_sh[row]) * y_ld;
#pragma unroll
        for (int n = 0; n < CN; ++n) {
          const int c = first + w0 + 32 * n + 2 * c16;
          if (c + 2 <= width) {
            const float2 now = {was[r][e][n].x + f * acc[r][n][0][e], was[r][e][n].y + f * acc[r][n][1][e]};
            __builtin_memcpy(y + c, &now, 8);
          } else if (c < width) {
            y[c] += f * acc[r][n][0][e];
          }
        }
      }
    }
    if constexpr (R == 1) break;
    if ((first += CB) >= last) break;
    load_b(0);
    load_y();
    __syncthreads();
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
  const float scale = a.scale[tile.adapter];
  const int row = a.order[tile.first + min(c16, tile.count - 1)];
  const uint16_t* const x = a.X + size_t(row) * a.x_ld + 8 * q4;
  const uint16_t* ar[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) ar[b] = a.A + (size_t(tile.adapter) * a.n_low + s * a.rank + min(16 * b + c16, a.rank - 1)) * a.D + 8 * q4;
  const uint16_t* const B = a.B + (size_t(tile.adapter) * a.n_out + b0) * a.rank;
  u32x4 xr[AHEAD], av[AHEAD][NB];
  const int steps = (max(0, a.D / 32 - wave) + 15) / 16;
  auto load = [&](int s0) {  // past the last, the last again
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int d = 32 * (wave + 16 * min(s0 + i, steps - 1));
#pragma unroll
      for (int b = 0; b < NB; ++b) av[i][b] = *reinterpret_cast<const u32x4*>(ar[b] + d);
      xr[i] = *reinterpret_cast<const u32x4*>(x + d);
    }
  };
  f32x4 acc[NB];
  float was[4][4];
  int64_t y_row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) y_row[i] = int64_t(a.order[tile.first + min(4 * q4 + i, tile.count - 1)]) * a.y_ld;
  float* const Y = a.Y + a.y_off[s];
  u32x4 bq[K / 32][4];
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x4{0, 0, 0, 0};
  if (steps > 0) load(0);
  // What the second product needs comes behind them. Columns behind the slice's end see its last again.
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int col = min(c0 + 16 * n + c16, width - 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) was[i][n] = Y[y_row[i] + col];
    const uint16_t* const of = B + size_t(col) * a.rank;
#pragma unroll
    for (int k = 0; k < K / 32; ++k) bq[k][n] = *reinterpret_cast<const u32x4*>(of + (32 * k + 8 * q4 < a.rank ? 32 * k + 8 * q4 : 0));
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
  f32x4 f = {scale, scale, scale, scale};
  if constexpr (DT == ESP_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= two_to(power_of(most[4 * q4 + i]));
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < K / 32; ++k)
#pragma unroll
      for (int t = 0; t < T; ++t) sum = mfma16x32<DT>(*reinterpret_cast<const u32x4*>(&low[t][c16][32 * k + 8 * q4]), bq[k][n], sum);
    mfma_settle(sum);
    const int col = c0 + 16 * n + c16;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * q4 + i < tile.count && col < width) Y[y_row[i] + col] = was[i][n] + f[i] * sum[i];
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
  constexpr int CB = R == 1 ? 256 : 128;
  int all = 0, blocks = 0;
  for (int s = 0; s < a.n_slices; ++s) all += (a.width[s] + CB - 1) / CB;
  const int each = lowrank_blocks_each(R, n_tiles, all);
  for (int s = 0; s < a.n_slices; ++s) blocks += (a.width[s] + CB * each - 1) / (CB * each);
  const dim3 up{unsigned(n_tiles + 7) / 8 * 8 * unsigned(blocks)};
  const size_t lds = size_t(DT == ESP_F16 ? 2 : 3) * 16 * R * ((a.rank + 31) / 32 * 32 + 8) * 2;
  if (R == 4 && a.rank <= 16) hipLaunchKernelGGL((lowrank_up_kernel<DT, 4, 16>), up, dim3(256), lds, st, a, n_tiles, blocks, each);
  else if (R == 4 && a.rank <= 32) hipLaunchKernelGGL((lowrank_up_kernel<DT, 4, 32>), up, dim3(256), lds, st, a, n_tiles, blocks, each);
  else if (a.rank <= 64) hipLaunchKernelGGL((lowrank_up_kernel<DT, R, 64>), up, dim3(256), lds, st, a, n_tiles, blocks, each);
  else hipLaunchKernelGGL((lowrank_up_kernel<DT, R, 128>), up, dim3(256), lds, st, a, n_tiles, blocks, each);
  return hipGetLastError();
}

template <int DT>
static hipError_t run_any(const LowRankArgs& a, int rows_per_tile, int n_tiles, hipStream_t st) {
  if (rows_per_tile != 16) return run_lowrank<DT, 4>(a, n_tiles, st);
  if (!lowrank_fused(a.D, a.rank, a.n_slices, a.width, n_tiles)) return run_lowrank<DT, 1>(a, n_tiles, st);
  if (a.rank <= 16) run_fused<DT, 1>(a, n_tiles, st);
  else run_fused<DT, 2>(a, n_tiles, st);
  return hipGetLastError();
}

hipError_t launch_lowrank(int dt, const LowRankArgs& a, int rows_per_tile, int n_tiles, hipStream_t st) {
  return dt == ESP_F16 ? run_any<ESP_F16>(a, rows_per_tile, n_tiles, st) : run_any<ESP_BF16>(a, rows_per_tile, n_tiles, st);
}

}  // namespace esp
