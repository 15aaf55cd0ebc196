// Linear attention with a decay for each head, or for each row and head: per head
//   S_t = exp(d_t) S_{t-1} + k_t^T v_t        (dk x dv, fp32, in slots that the caller keeps)
//   o_t = scale q_t S_t
// Two kernels, one for sequences of few rows (a decode step's single tokens, drafts) and one for prompts.
#include "common.hpp"
#include "lds_direct.hpp"
#include "linear_shape.hpp"

namespace esp {

namespace {

// A log decay in log2 units as the kernels take it: never above 0, and not below what makes the factor 0 in fp32 anyway. NaN stays.
__device__ __forceinline__ float decay_log2(float d) {
  const float x = d * kLog2e;
  return x > 0.0f ? 0.0f : x < -200.0f ? -200.0f : x;
}

// ---- few rows -----------------------------------------------------------------------------------------------------------
// The recurrence as it stands. Bound by HBM: a state is read and written once, 4 dk dv bytes each way, and all that is done to it between
// is 4 dk dv operations a row. A workgroup takes DVB columns of one state: lane l of a row group four columns, the row groups every RG-th
// row of the state, all loads out before the first use. A row's outputs are summed over the lane's rows, over the wavefront by exchanges
// and over the four wavefronts through LDS at the end, for all rows of the sequence at once.
template <int DT, int DVB, int DK>
__global__ __launch_bounds__(256) void linear_few_kernel(const LinearArgs a) {
  constexpr int LPR = DVB / 4, RG = 256 / LPR, NK = DK / RG;
  __shared__ float qk[2][kLinearFew][DK];
  __shared__ __attribute__((aligned(16))) float out[kLinearFew][4][DVB];
  const int blocks = a.dv / DVB, h = blockIdx.x / blocks, c0 = (blockIdx.x - h * blocks) * DVB;
  const esp_linear_tile tile = a.tiles[blockIdx.y];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = c0 + 4 * int(threadIdx.x % LPR), g = threadIdx.x / LPR;
  const size_t at = size_t(h) * DK * a.dv + col, slot = size_t(a.H) * DK * a.dv;
  f32x4 s[NK];
  if (tile.src >= 0) {
    const float* from = a.states + size_t(tile.src) * slot + at;
#pragma unroll
    for (int i = 0; i < NK; ++i) s[i] = *reinterpret_cast<const f32x4*>(from + size_t(g + RG * i) * a.dv);
  } else {
#pragma unroll
    for (int i = 0; i < NK; ++i) s[i] = f32x4{0, 0, 0, 0};
  }
  const int kh = h / a.group;
  for (int i = threadIdx.x; i < tile.rows * (DK / 2); i += 256) {
    const int m = i / (DK / 2), d = 2 * (i - m * (DK / 2));
    const uint32_t q = *reinterpret_cast<const uint32_t*>(a.Q + size_t(tile.row0 + m) * a.q_ld + size_t(kh) * DK + d);
    const uint32_t k = *reinterpret_cast<const uint32_t*>(a.K + size_t(tile.row0 + m) * a.k_ld + size_t(kh) * DK + d);
    qk[0][m][d] = unpack_lo<DT>(q);
    qk[0][m][d + 1] = unpack_hi<DT>(q);
    qk[1][m][d] = unpack_lo<DT>(k);
    qk[1][m][d + 1] = unpack_hi<DT>(k);
  }
  __syncthreads();
  for (int m = 0; m < tile.rows; ++m) {
    const int row = tile.row0 + m;
    const float f = fast_exp2(decay_log2(a.decay[size_t(row) * a.decay_ld + h]));
    const u32x2 vb = *reinterpret_cast<const u32x2*>(a.V + size_t(row) * a.v_ld + size_t(h) * a.dv + col);
    const f32x4 v = {unpack_lo<DT>(vb.x), unpack_hi<DT>(vb.x), unpack_lo<DT>(vb.y), unpack_hi<DT>(vb.y)};
    f32x4 o = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < NK; ++i) {
      const float q = qk[0][m][g + RG * i], k = qk[1][m][g + RG * i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[i][e] = __builtin_fmaf(k, v[e], s[i][e] * f);
        o[e] = __builtin_fmaf(q, s[i][e], o[e]);
      }
    }
#pragma unroll
    for (int x = LPR; x < 64; x <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
    if (lane < LPR) *reinterpret_cast<f32x4*>(&out[m][wave][4 * lane]) = o;
  }
  if (tile.dst >= 0) {
    float* to = a.states + size_t(tile.dst) * slot + at;
#pragma unroll
    for (int i = 0; i < NK; ++i) *reinterpret_cast<f32x4*>(to + size_t(g + RG * i) * a.dv) = s[i];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tile.rows * LPR; i += 256) {
    const int m = i / LPR, c = 4 * (i - m * LPR);
    f32x4 o = *reinterpret_cast<const f32x4*>(&out[m][0][c]);
#pragma unroll
    for (int w = 1; w < 4; ++w) o += *reinterpret_cast<const f32x4*>(&out[m][w][c]);
    o *= a.scale;
    *reinterpret_cast<u32x2*>(a.O + size_t(tile.row0 + m) * a.o_ld + size_t(h) * a.dv + c0 + c) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
  }
}

// ---- many rows ----------------------------------------------------------------------------------------------------------
// 64 rows at a time. With c_i the sum of the chunk's log decays up to row i, C its last, and S the state in front of it,
//   O_i = exp(c_i) q_i S + sum_{j <= i} exp(c_i - c_j) (q_i . k_j) v_j
//   S'  = exp(C) S + sum_j k_j^T (exp(C - c_j) v_j)
// which are four matrix products: P = Q K^T, Q S, P V and K^T V'. One workgroup takes one head's DVB columns of V; wavefront w owns 32 of
// them, the state's among them, which never leave its registers: as the result of K^T V' a lane holds 8 consecutive rows (dk) of one column
// of S in a row of registers (the rows of K^T are asked for in an order that makes it so), which is how it has to hold them as an operand
// of (Q S)^T. P is shared: every wavefront makes its rows of it and they meet in LDS.
//
// What is rounded to 16 bits on the way into a product enters as the sum of several such numbers, since sums of products with signs
// would keep each one's error beside results that the state holds in fp32: S and P as two (16 bits or more, like the output), V' as two
// of 11 (fp16) or three of 8 bits (bf16), for which the state's own error is that of fp32. fp16 parts are scaled by powers of two, S by
// one a wavefront, P by one a row, V' by one a column: they lose what lies 2^-39 below the largest.
//
// A sequence may be cut into segments: a first launch makes each segment's own state from zero (STATE; the first one's from
// the sequence's), and the segments then start from the sum of those in front of them, each decayed over the segments between.

using lds_u32x4 = const __attribute__((address_space(3))) u32x4;
using lds_u32x4_out = __attribute__((address_space(3))) u32x4;
using lds_u32x2_out = __attribute__((address_space(3))) u32x2;

constexpr int kPBytes = 32 * 64 + 32 * 128;  // rows 0 .. 31 of P have no weights behind column 31

// LDS of the chunked kernel, bytes. Rows of Q and K in memory order, 16-byte parts turned by the row; K^T and V^T [dk or dv][64 rows].
template <int DK, int DVB, bool STATE>
struct ChunkLds {
  static constexpr int kQ = 0;
  static constexpr int kK = STATE ? 0 : 64 * DK * 2;
  static constexpr int kKT = STATE ? 0 : 2 * 64 * DK * 2;
  static constexpr int kVT = kKT + 64 * DK * 2;
  static constexpr int kP = kVT + 64 * DVB * 2;             // two numbers for each weight
  static constexpr int kCum = kP + (STATE ? 0 : 2 * kPBytes);  // double[64]: c
  static constexpr int kLeft = kCum + 512;                  // float[64]: exp(C - c_j)
  static constexpr int kRowF = kLeft + 256;                 // float[64]: exp(c_i)
  static constexpr int kPInv = kRowF + 256;                 // float[64]: what undoes P's scale
  static constexpr int kTotal = kPInv + 256;                // float: exp(C)
  static constexpr int kBytes = kTotal + 256;
};

// Parts of rows of DK numbers and of rows of 64 (K^T, V^T, P): where part c of row r lies.
template <int DK>
__device__ __forceinline__ int row_part(int r, int c) {
  return r * (DK * 2) + ((DK == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7)) << 4);
}
__device__ __forceinline__ int col_part(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7) ^ ((r >> 3) & 2)) << 4); }

__device__ __forceinline__ int p_part(int r, int c) {
  return r < 32 ? r * 64 + ((c ^ ((r >> 2) & 3)) << 4) : 2048 + (r - 32) * 128 + ((c ^ ((r >> 1) & 7)) << 4);
}

// 2^(14 - e) for a value of exponent e, and its inverse: the power of two that brings the largest of a set of numbers just below
// fp16's largest. At most 2^most (126 or less); both are normal numbers.
__device__ __forceinline__ void scale_for(float largest, int most, float& up, float& down) {
  uint32_t e = (__builtin_bit_cast(uint32_t, largest) >> 23) & 255;
  e = max(e, uint32_t(141 - most));
  up = __builtin_bit_cast(float, (268 - e) << 23);
  down = __builtin_bit_cast(float, (e - 14) << 23);
}

// Where the sums are an fp16 output's, no scale above 2^60: what that leaves below fp16's grid, 2^-85, is nothing beside an output's own
// step, and the other half of the sums, which takes the same scale, stays far from fp32's largest.
constexpr int kOutputScale = 60;

// 8 numbers as N numbers of 16 bits each.
template <int DT, int N>
__device__ __forceinline__ void split8(const float (&x)[8], u32x4 (&out)[N]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float lo = x[2 * e], hi = x[2 * e + 1];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const uint32_t w = pack2<DT>(lo, hi);
      out[n][e] = w;
      if (n + 1 < N) {
        lo -= unpack_lo<DT>(w);
        hi -= unpack_hi<DT>(w);
      }
    }
  }
}

__device__ __forceinline__ float abs_max_halves(float x) { return fmaxf(x, __shfl_xor(x, 32)); }

template <int DT, int DK, int DVB, bool STATE>
__global__ __launch_bounds__(2 * DVB, DK == 128 && DVB == 64 ? 1 : 2) void linear_chunk_kernel(const LinearArgs a) {
  constexpr int NW = DVB / 32, T = 64 * NW, KT = DK / 32, NV = DT == ESP_F16 ? 2 : 3;
  using L = ChunkLds<DK, DVB, STATE>;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const esp_linear_tile tile = a.tiles[blockIdx.y];
  if (STATE && tile.after == 0) return;
  const int blocks = a.dv / DVB, h = blockIdx.x / blocks, blk = blockIdx.x - h * blocks;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hb = lane >> 5;
  const int dv0 = h * a.dv + blk * DVB;  // first column of V and O
  const int kh = h / a.group;
  const int col = blk * DVB + 32 * wave + l32;  // this lane's column of the state
  const size_t slot = size_t(a.H) * DK * a.dv;
  double* const cum = reinterpret_cast<double*>(lds + L::kCum);
  float* const left = reinterpret_cast<float*>(lds + L::kLeft);
  float* const rowf = reinterpret_cast<float*>(lds + L::kRowF);
  float* const pinv = reinterpret_cast<float*>(lds + L::kPInv);
  float* const total = reinterpret_cast<float*>(lds + L::kTotal);

  // ---- the state in front of the segment
  f32x16 S[KT];
  const size_t rec_at = ((size_t(h) * blocks + blk) * NW + wave) * (size_t(KT) * 16 * 64) + size_t(lane) * 4;
  auto record = [&](int i) { return a.parts + size_t(i) * slot + rec_at; };
  // Register 4 i + e of tile t: row 32 t + 16 (i / 2) + 8 hb + 4 (i % 2) + e of the column.
  auto state_at = [&](int t, int i) { return size_t(h) * DK * a.dv + size_t(32 * t + 16 * (i >> 1) + 8 * hb + 4 * (i & 1)) * a.dv + col; };
#pragma unroll
  for (int t = 0; t < KT; ++t) S[t] = f32x16{};
  if (tile.before == 0) {
    if (tile.src >= 0 && !(tile.part >= 0 && !STATE)) {
      const float* from = a.states + size_t(tile.src) * slot;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[t][4 * i + e] = from[state_at(t, i) + size_t(e) * a.dv];
    } else if (tile.src >= 0) {  // the first launch has copied it: the last segment may be writing the slot by now
      const float* from = record(tile.part);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(from + (t * 4 + i) * 256);
#pragma unroll
          for (int e = 0; e < 4; ++e) S[t][4 * i + e] = x[e];
        }
    }
  } else if (!STATE) {
    double since = 0.0;  // log2 of the decays of the segments between
    for (int j = tile.before; j >= 1; --j) {
      const float f = fast_exp2(float(since));
      const float* from = record(tile.part + j);
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(from + (t * 4 + i) * 256);
#pragma unroll
          for (int e = 0; e < 4; ++e) S[t][4 * i + e] = __builtin_fmaf(x[e], f, S[t][4 * i + e]);
        }
      since += a.part_totals[size_t(tile.part + j) * a.H + h];
    }
  }
  auto keep_record = [&](int r) {
    float* to = record(r);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(to + (t * 4 + i) * 256) = f32x4{S[t][4 * i], S[t][4 * i + 1], S[t][4 * i + 2], S[t][4 * i + 3]};
  };
  if (STATE && tile.before == 0 && tile.src >= 0) keep_record(tile.part);

  // ---- chunks: 4 rows x 8 columns a thread and piece of K, Q and V on their way to LDS
  constexpr int NI = STATE ? (2 * DK + T - 1) / T : (4 * DK) / T, kParts = DK / 8, vParts = DVB / 8;
  u32x4 kq[NI][4], vv[4];
  const float g_const = a.decay_ld ? 0.0f : decay_log2(a.decay[h]);
  float g_row = 0.0f;
  const int n_chunks = (tile.rows + 63) >> 6;
  auto fetch = [&](int c) __attribute__((always_inline)) {
    const int r0 = tile.row0 + 64 * c, last = tile.row0 + tile.rows - 1;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int it = tid + T * n;
      if (STATE && it >= 2 * DK) break;
      const bool isK = STATE || it < 2 * DK;
      const int b = isK ? it : it - 2 * DK, r = r0 + 4 * (b / kParts), part = b % kParts;
      const uint16_t* from = (isK ? a.K : a.Q) + size_t(kh) * DK + 8 * part;
      const size_t ld = isK ? a.k_ld : a.q_ld;
#pragma unroll
      for (int i = 0; i < 4; ++i) kq[n][i] = *reinterpret_cast<const u32x4*>(from + size_t(min(r + i, last)) * ld);
    }
    const int r = r0 + 4 * (tid / vParts), part = tid % vParts;
#pragma unroll
    for (int i = 0; i < 4; ++i) vv[i] = *reinterpret_cast<const u32x4*>(a.V + size_t(min(r + i, last)) * a.v_ld + dv0 + 8 * part);
    if (a.decay_ld) g_row = decay_log2(a.decay[size_t(min(r0 + lane, last)) * a.decay_ld + h]);
  };
  // Rows behind the segment's last are zeros in K and V.
  auto clear_past = [&](u32x4 (&x)[4], int r, int n) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r + i >= n) x[i] = u32x4{0, 0, 0, 0};
  };
  // Operands' places: one address each, the parts of a row by turning bits of it, tiles behind each other as the instruction's own offset.
  // Worked out again in every chunk: kept for the next they would be spilled.
  const uint32_t base = uint32_t(uintptr_t(lds));
  auto place = [&](int at) {
    uint32_t x = base + uint32_t(at);
    asm volatile("" : "+v"(x));
    return x;
  };
  auto read = [&](uint32_t at) { return *reinterpret_cast<lds_u32x4*>(at); };
  // 4 rows of 8 columns, rows 4 group .. + 3 and their part: as they come, and as 8 columns of 4 rows into a [columns][64 rows] array.
  auto put_rows = [&](const u32x4 (&x)[4], int to, int group, int part) __attribute__((always_inline)) {
    const uint32_t at = place(to + row_part<DK>(4 * group, part));
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<lds_u32x4_out*>((at ^ ((DK == 128 ? j : j >> 1) << 4)) + j * (DK * 2)) = x[j];
  };
  auto put_columns = [&](const u32x4 (&x)[4], int to, int group, int part) __attribute__((always_inline)) {
    const uint32_t at = place(to + col_part(8 * part, group >> 1) + 8 * (group & 1));
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t sel = s ? 0x07060302u : 0x05040100u;
        *reinterpret_cast<lds_u32x2_out*>((at ^ (p << 4)) + (2 * p + s) * 128) =
            u32x2{__builtin_amdgcn_perm(x[1][p], x[0][p], sel), __builtin_amdgcn_perm(x[3][p], x[2][p], sel)};
      }
  };

  if (n_chunks > 0) fetch(0);
  double so_far = 0.0;
  for (int c = 0; c < n_chunks; ++c) {
    const int n = min(64, tile.rows - 64 * c);
    if (c > 0) __syncthreads();  // everybody is done with the chunk in front of this one
    if (n < 64) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int it = tid + T * i;
        if (STATE || it < 2 * DK) clear_past(kq[i], 4 * (it / kParts), n);
      }
      clear_past(vv, 4 * (tid / vParts), n);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int it = tid + T * i;
      if (STATE && it >= 2 * DK) break;
      const bool isK = STATE || it < 2 * DK;
      const int b = isK ? it : it - 2 * DK;
      if (!STATE) put_rows(kq[i], isK ? L::kK : L::kQ, b / kParts, b % kParts);
      if (isK) put_columns(kq[i], L::kKT, b / kParts, b % kParts);
    }
    put_columns(vv, L::kVT, tid / vParts, tid % vParts);
    double cl;  // C, in every wavefront
    {
      double s;
      if (a.decay_ld) {
        s = lane < n ? double(g_row) : 0.0;
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) {
          const double up = __shfl_up(s, x);
          s += lane >= x ? up : 0.0;
        }
      } else {
        s = double(g_const) * min(lane + 1, n);
      }
      cl = __shfl(s, 63);
      if (wave == 0) {
        cum[lane] = s;
        left[lane] = lane < n ? fast_exp2(float(cl - s)) : 0.0f;
        rowf[lane] = fast_exp2(float(s));
        if (lane == 0) *total = fast_exp2(float(cl));
      }
    }
    so_far += cl;
    __syncthreads();
    if (STATE && c + 1 < n_chunks) fetch(c + 1);

    f32x16 O[2];
    float s_down = 1.0f;
    if constexpr (!STATE) {
      // P^T, 16 x 16 at a time: lane l has row 16 rt + l % 16 and columns 16 jt + 4 (l / 16) .. + 3.
      const int l16 = lane & 15, q4 = lane >> 4;
#pragma unroll
      for (int half = 0; half < (NW == 4 ? 1 : 2); ++half) {
        const int rt = NW == 4 ? wave : half ? 3 - wave : wave;
        const int row = 16 * rt + l16;
        u32x4 qf[DK / 32];
        const uint32_t q_at = place(L::kQ + row_part<DK>(row, q4)), k_at = place(L::kK + row_part<DK>(l16, q4));
#pragma unroll
        for (int kk = 0; kk < DK / 32; ++kk) qf[kk] = read(q_at ^ (kk << 6));
        const double ci = cum[row];
        float x[4][4], mx = 0.0f;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[jt][e] = 0.0f;
          if (jt > rt) continue;
          f32x4 acc = {0, 0, 0, 0};
#pragma unroll
          for (int kk = 0; kk < DK / 32; ++kk) acc = mfma16x32<DT>(read((k_at ^ (kk << 6)) + jt * (32 * DK)), qf[kk], acc);
          mfma_settle(acc);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int j = 16 * jt + 4 * q4 + e;
            const float w = fast_exp2(float(ci - cum[j]));
            x[jt][e] = j <= row ? acc[e] * w : 0.0f;
            mx = fmaxf(mx, fabsf(x[jt][e]));
          }
        }
        if constexpr (DT == ESP_F16) {
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          float up, down;
          scale_for(mx, kOutputScale, up, down);
#pragma unroll
          for (int jt = 0; jt < 4; ++jt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[jt][e] *= up;
          if (q4 == 0) pinv[row] = down;
        }
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          if (jt > (rt | 1)) continue;  // (the product reads columns in groups of 32)
          const uint32_t w0 = pack2<DT>(x[jt][0], x[jt][1]), w1 = pack2<DT>(x[jt][2], x[jt][3]);
          const uint32_t r0 = pack2<DT>(x[jt][0] - unpack_lo<DT>(w0), x[jt][1] - unpack_hi<DT>(w0));
          const uint32_t r1 = pack2<DT>(x[jt][2] - unpack_lo<DT>(w1), x[jt][3] - unpack_hi<DT>(w1));
          const int to = L::kP + p_part(row, 2 * jt + (q4 >> 1)) + 8 * (q4 & 1);
          *reinterpret_cast<u32x2*>(lds + to) = u32x2{w0, w1};
          *reinterpret_cast<u32x2*>(lds + to + kPBytes) = u32x2{r0, r1};
        }
      }
      // (Q S)^T
      O[0] = f32x16{};
      O[1] = f32x16{};
      float s_up = 1.0f;
      if constexpr (DT == ESP_F16) {
        float mx = 0.0f;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) mx = fmaxf(mx, fabsf(S[t][e]));
        if (__builtin_expect(__any(mx == INFINITY), 0)) {  // infinities are not what the others are scaled by
          mx = 0.0f;
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fabsf(S[t][e]) < INFINITY ? fmaxf(mx, fabsf(S[t][e])) : mx;
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) mx = fmaxf(mx, __shfl_xor(mx, x));
        scale_for(mx, kOutputScale, s_up, s_down);
      }
      const uint32_t q_at = place(L::kQ + row_part<DK>(l32, hb));
#pragma unroll
      for (int ks = 0; ks < DK / 16; ++ks) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = DT == ESP_F16 ? S[ks >> 1][8 * (ks & 1) + e] * s_up : S[ks >> 1][8 * (ks & 1) + e];
        u32x4 sp[2];
        split8<DT, 2>(x, sp);
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
          const u32x4 q = read((q_at ^ (ks << 5)) + rt * (64 * DK));
          O[rt] = mfma32x16<DT>(sp[0], q, O[rt]);
          O[rt] = mfma32x16<DT>(sp[1], q, O[rt]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (c + 1 < n_chunks) fetch(c + 1);
      __syncthreads();  // P is there, and nobody reads Q and K any more
    }
    u32x4 vr[4];
    auto read_v = [&] {
      const uint32_t v_at = place(L::kVT + col_part(32 * wave + l32, hb));
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) vr[ks] = read(v_at ^ (ks << 5));
    };
    read_v();
    if constexpr (!STATE) {
      // An infinite or NaN value may not reach the rows in front of its own, whose weight of it is zero.
      float nf = 0.0f;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int e = 0; e < 4; ++e) nf = fmaf(unpack_lo<DT>(vr[ks][e]), 0.0f, fmaf(unpack_hi<DT>(vr[ks][e]), 0.0f, nf));
      const bool odd = __any(nf != 0.0f);
      if (__builtin_expect(odd, 0)) {
        constexpr uint32_t ex = DT == ESP_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t w = vr[ks][e];
            vr[ks][e] = w & (((w & ex) == ex ? 0u : 0xffffu) | ((w >> 16 & ex) == ex ? 0u : 0xffff0000u));
          }
      }
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const int row = 32 * rt + l32;
        mfma_settle(O[rt]);
        float f = rowf[row];
        if constexpr (DT == ESP_F16) {
          const float d = pinv[row];  // (a power of two)
          f *= s_down;
          O[rt] *= f;
          O[rt] *= 1.0f / d;
        } else {
          O[rt] *= f;
        }
        const uint32_t p_at = place(L::kP + p_part(row, hb));
#pragma unroll
        for (int ks = 0; ks < 2 + 2 * rt; ++ks) {
          O[rt] = mfma32x16<DT>(vr[ks], read(p_at ^ (ks << 5)), O[rt]);
          O[rt] = mfma32x16<DT>(vr[ks], read((p_at ^ (ks << 5)) + kPBytes), O[rt]);
        }
        mfma_settle(O[rt]);
        if (__builtin_expect(odd, 0)) {
          // Rows 8 (e / 4) + 4 hb + e % 4 of the wavefront's part of V^T: their turns differ by constants.
#pragma unroll 1
          for (int j = 0; j <= row; ++j) {
            const float p = unpack_lo<DT>(*reinterpret_cast<const uint16_t*>(lds + L::kP + p_part(row, j >> 3) + 2 * (j & 7)));
            const uint32_t at = place(L::kVT + (32 * wave + 4 * hb) * 128 + (((j >> 3) ^ (2 * hb)) << 4) + 2 * (j & 7));
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              constexpr auto turn = [](int d) { return ((d >> 1) & 7) ^ ((d >> 3) & 2); };
              const int d = 8 * (e >> 2) + (e & 3);
              const float v = unpack_lo<DT>(*reinterpret_cast<const __attribute__((address_space(3))) uint16_t*>((at ^ (turn(d) << 4)) + d * 128));
              if (!(fabsf(v) < INFINITY)) O[rt][e] += p * v;
            }
          }
        }
        O[rt] *= DT == ESP_F16 ? pinv[row] * a.scale : a.scale;
      }
      if (__builtin_expect(odd, 0)) read_v();
      // Through LDS, where Q and K were, a wavefront's 64 rows of 64 bytes each; 16-byte parts turned by the row.
      char* const mine = lds + L::kQ + wave * 4096;
      auto part_at = [&](int r, int p) { return mine + r * 64 + ((p ^ ((r >> 2) & 3)) << 4); };
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x2*>(part_at(32 * rt + l32, i) + 8 * hb) =
              u32x2{pack2<DT>(O[rt][4 * i], O[rt][4 * i + 1]), pack2<DT>(O[rt][4 * i + 2], O[rt][4 * i + 3])};
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 16 * i + (lane >> 2), p = lane & 3;
        const u32x4 x = *reinterpret_cast<const u32x4*>(part_at(r, p));
        if (r < n) *reinterpret_cast<u32x4*>(a.O + size_t(tile.row0 + 64 * c + r) * a.o_ld + dv0 + 32 * wave + 8 * p) = x;
      }
    }
    // S = exp(C) S + K^T V'. (The state behind the segment is of use only where somebody reads it.)
    if (STATE || c + 1 < n_chunks || tile.dst >= 0) {
      const float f = *total;
      const uint32_t k_at = place(L::kKT + col_part(swap23(l32), hb));
      auto weighted = [&](int ks, float (&x)[8]) __attribute__((always_inline)) {
        const f32x4 w0 = *reinterpret_cast<const f32x4*>(left + 16 * ks + 8 * hb), w1 = *reinterpret_cast<const f32x4*>(left + 16 * ks + 8 * hb + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = unpack_lo<DT>(vr[ks][e]) * (e < 2 ? w0 : w1)[2 * (e & 1)];
          x[2 * e + 1] = unpack_hi<DT>(vr[ks][e]) * (e < 2 ? w0 : w1)[2 * (e & 1) + 1];
        }
      };
      if constexpr (DT == ESP_F16) {
        float mx = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          float x[8];
          weighted(ks, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[e]));
        }
        mx = abs_max_halves(mx);
        float up, down;
        scale_for(mx, 126, up, down);
        u32x4 vs[4][NV];
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          float x[8];
          weighted(ks, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= up;
          split8<DT, NV>(x, vs[ks]);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          f32x16 d{};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const u32x4 k = read((k_at ^ (ks << 5)) + t * 4096);
#pragma unroll
            for (int v = 0; v < NV; ++v) d = mfma32x16<DT>(k, vs[ks][v], d);
          }
          mfma_settle(d);
#pragma unroll
          for (int e = 0; e < 16; ++e) S[t][e] = __builtin_fmaf(d[e], down, S[t][e] * f);
        }
      } else {
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] *= f;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          float x[8];
          weighted(ks, x);
          u32x4 vs[NV];
          split8<DT, NV>(x, vs);
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            const u32x4 k = read((k_at ^ (ks << 5)) + t * 4096);
#pragma unroll
            for (int v = 0; v < NV; ++v) S[t] = mfma32x16<DT>(k, vs[v], S[t]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) mfma_settle(S[t]);
      }
    }
  }

  if (STATE) {
    keep_record(tile.part + 1 + tile.before);
    if (tid == 0 && blk == 0) a.part_totals[size_t(tile.part + 1 + tile.before) * a.H + h] = so_far;
  } else if (tile.dst >= 0) {
    float* to = a.states + size_t(tile.dst) * slot;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[state_at(t, i) + size_t(e) * a.dv] = S[t][4 * i + e];
  }
}

template <int DT, int DK, int DVB, bool STATE>
hipError_t launch_chunk(const LinearArgs& a, const esp_linear_tile* tiles, int n, hipStream_t st) {
  constexpr auto k = linear_chunk_kernel<DT, DK, DVB, STATE>;
  constexpr size_t smem = ChunkLds<DK, DVB, STATE>::kBytes;
  const hipError_t e = allow_dynamic_lds<k>(smem);
  if (e != hipSuccess) return e;
  LinearArgs b = a;
  b.tiles = tiles;
  hipLaunchKernelGGL(k, dim3(unsigned(a.H * (a.dv / DVB)), unsigned(n)), dim3(2 * DVB), smem, st, b);
  return hipGetLastError();
}

template <int DT, int DK, int DVB>
hipError_t launch_chunks(const LinearArgs& a, const esp_linear_tile* tiles, int n, bool split, hipStream_t st) {
  const hipError_t e = split ? launch_chunk<DT, DK, DVB, true>(a, tiles, n, st) : hipSuccess;
  return e == hipSuccess ? launch_chunk<DT, DK, DVB, false>(a, tiles, n, st) : e;
}

template <int DT, int DVB, int DK>
hipError_t launch_few_t(const LinearArgs& a, int n, hipStream_t st) {
  hipLaunchKernelGGL((linear_few_kernel<DT, DVB, DK>), dim3(unsigned(a.H * (a.dv / DVB)), unsigned(n)), dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int DT, int DK>
hipError_t launch_few(const LinearArgs& a, int n, hipStream_t st) {
  if (a.dv % 128 == 0 && long(a.H) * (a.dv / 128) * n >= 4 * kComputeUnits) return launch_few_t<DT, 128, DK>(a, n, st);
  if (long(a.H) * (a.dv / 64) * n >= 4 * kComputeUnits) return launch_few_t<DT, 64, DK>(a, n, st);
  return launch_few_t<DT, 32, DK>(a, n, st);
}

template <int DT, int DK>
hipError_t launch_t(const LinearArgs& a, int n_few, int n_chunked, bool split, hipStream_t st) {
  hipError_t e = n_few > 0 ? launch_few<DT, DK>(a, n_few, st) : hipSuccess;
  if (e != hipSuccess || n_chunked <= 0) return e;
  if (linear_cols(a.dv) == 128) return launch_chunks<DT, DK, 128>(a, a.tiles + n_few, n_chunked, split, st);
  return launch_chunks<DT, DK, 64>(a, a.tiles + n_few, n_chunked, split, st);
}

template <int DT, int DK, int DVB>
hipError_t allow_chunk() {
  const hipError_t e = allow_dynamic_lds<linear_chunk_kernel<DT, DK, DVB, true>>(ChunkLds<DK, DVB, true>::kBytes);
  return e == hipSuccess ? allow_dynamic_lds<linear_chunk_kernel<DT, DK, DVB, false>>(ChunkLds<DK, DVB, false>::kBytes) : e;
}

template <int DT>
hipError_t allow_chunks() {
  hipError_t e = allow_chunk<DT, 64, 64>();
  if (e == hipSuccess) e = allow_chunk<DT, 64, 128>();
  if (e == hipSuccess) e = allow_chunk<DT, 128, 64>();
  if (e == hipSuccess) e = allow_chunk<DT, 128, 128>();
  return e;
}

}  // namespace

hipError_t linear_init_attributes() {
  const hipError_t e = allow_chunks<ESP_F16>();
  return e == hipSuccess ? allow_chunks<ESP_BF16>() : e;
}

// Tiles: n_few of the recurrent kernel, then n_chunked; at most 65535 of each, and the dims are served: the caller has checked.
hipError_t launch_linear(int dt, const LinearArgs& a, int n_few, int n_chunked, bool split, hipStream_t st) {
  if (dt == ESP_F16) return a.dk == 64 ? launch_t<ESP_F16, 64>(a, n_few, n_chunked, split, st) : launch_t<ESP_F16, 128>(a, n_few, n_chunked, split, st);
  return a.dk == 64 ? launch_t<ESP_BF16, 64>(a, n_few, n_chunked, split, st) : launch_t<ESP_BF16, 128>(a, n_few, n_chunked, split, st);
}

}  // namespace esp
