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
// and over the four wavefronts through LDS at the end, for all rows of the sequence at once. 64 single tokens, 32 heads of 128 x 128: 54 us for
// 270 MB of states that come from HBM, 5.0 TB/s where a copy of as much reaches 5.4. A row costs 1.4 us of those on top.
template <int DT, int DVB, int DK>
__global__ __launch_bounds__(256) void linear_few_kernel(const LinearArgs a) {
  constexpr int LPR = DVB / 4, RG = 256 / LPR, NK = DK / RG;
  __shared__ float qk[2][kLinearFew][DK];
  __shared__ __attribute__((aligned(16))) float out[kLinearFew][4][DVB];
  const int blocks = a.dv / DVB, h = blockIdx.x / blocks, c0 = (blockIdx.x - h * blocks) * DVB;
  const esp_linear_tile tile = a.tiles[blockIdx.y];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = min(tile.rows, kLinearFew);
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
  for (int i = threadIdx.x; i < rows * (DK / 2); i += 256) {
    const int m = i / (DK / 2), d = 2 * (i - m * (DK / 2));
    const uint32_t q = *reinterpret_cast<const uint32_t*>(a.Q + size_t(tile.row0 + m) * a.q_ld + size_t(kh) * DK + d);
    const uint32_t k = *reinterpret_cast<const uint32_t*>(a.K + size_t(tile.row0 + m) * a.k_ld + size_t(kh) * DK + d);
    qk[0][m][d] = unpack_lo<DT>(q);
    qk[0][m][d + 1] = unpack_hi<DT>(q);
    qk[1][m][d] = unpack_lo<DT>(k);
    qk[1][m][d + 1] = unpack_hi<DT>(k);
  }
  __syncthreads();
  for (int m = 0; m < rows; ++m) {
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
  for (int i = threadIdx.x; i < rows * LPR; i += 256) {
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
// Bound by the matrix units and what feeds them: with the numbers counted a chunk of 64 rows, 128 x 128, is 13.6 million operations, 2 us of
// a compute unit's matrix units; two workgroups beside each other take 6.9 us for one each. 40 heads of 4 x 2048 rows, 128 x 128, bf16: 133 to 137 us;
// 32 heads of 16000 rows, 64 x 128, on 8 heads of Q and K: 146 to 152 us, in 16 segments. 539 and 655 MB move in
// that, at 4.0 and 4.4 TB/s, but they are the lesser part of what bounds it: the same passes with one head of Q and K for all heads, which is half of
// the first one's bytes, take 17 % and 5 % less.
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
  static constexpr int kLeft = kP + (STATE ? 0 : 2 * kPBytes);  // float[64]: exp(C - c_j)
  static constexpr int kRowF = kLeft + 256;                 // float[64]: scale exp(c_i)
  static constexpr int kTotal = kRowF + 256;                // float: exp(C)
  static constexpr int kColF = kTotal + 16;                 // float[4][64]: exp(b_t - c_j), b_t the sum in front of row 16 t, of the rows there
  static constexpr int kSince = kColF + (STATE ? 0 : 1024); // float[64][2]: c_i - b of the row's tile, in two numbers
  static constexpr int kPInv = kSince + (STATE ? 0 : 512);  // float[64]: what undoes P's scale
  static constexpr int kNone = kPInv + (STATE ? 0 : 256);               // where what has no place in P goes, a wavefront's over another's
  static constexpr int kBytes = kNone + (STATE ? 0 : 512);
};

// Parts of rows of DK numbers and of rows of 64 (K^T, V^T, P): where part c of row r lies.
template <int DK>
__device__ __forceinline__ int row_part(int r, int c) {
  return r * (DK * 2) + ((DK == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7)) << 4);
}
// (Of a read of 16 bytes a lane 16 lanes go at a time, one set those of rows 0 .. 3, 12 .. 15, 20 .. 27 of 32, the other the rest; written are eight
// columns 8 apart. Both find different places this way.)
__device__ __forceinline__ int col_part(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7) ^ ((r >> 4) & 3)) << 4); }

// Which 4 rows and which part of them piece b of a [64 rows][8 PARTS numbers] array is, such that 16 lanes one after the other hold 8 parts of
// 8 rows: as 8 bytes each in the columns of such an array that is all of LDS's banks once.
template <int PARTS>
__device__ __forceinline__ int piece_group(int b) {
  return PARTS == 16 ? ((b >> 5) << 1) | ((b >> 3) & 1) : b / PARTS;
}
template <int PARTS>
__device__ __forceinline__ int piece_part(int b) {
  return PARTS == 16 ? (b & 7) | ((b >> 1) & 8) : b % PARTS;
}

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

// 8 numbers times `by` (1 for bf16) as N numbers of 16 bits each.
template <int DT, int N>
__device__ __forceinline__ void split8(const float (&x)[8], float by, u32x4 (&out)[N]) {
  if constexpr (DT == ESP_F16) {
    static_assert(N == 2);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f16x2 a, b;
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // (an instruction each, which rounds its product or difference to fp16)
        a[i] = (_Float16)__builtin_fmaf(x[2 * e + i], by, 0.0f);
        b[i] = (_Float16)__builtin_fmaf(x[2 * e + i], by, -float(a[i]));
      }
      out[0][e] = __builtin_bit_cast(uint32_t, a);
      out[1][e] = __builtin_bit_cast(uint32_t, b);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float lo = x[2 * e], hi = x[2 * e + 1];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t w = pack2<DT>(lo, hi);
      if (n + 1 < N) asm("" : "+v"(w));  // (left alone the compiler converts the lower one once more instead of shifting it out)
      out[n][e] = w;
      if (n + 1 < N) {
        lo -= unpack_lo<DT>(w);
        hi -= unpack_hi<DT>(w);
      }
    }
  }
}

// acc + the two storage elements of a dword times zero: NaN where one of them is not finite.
template <int DT>
__device__ __forceinline__ float times_zero2(uint32_t w, float acc) {
  if constexpr (DT == ESP_F16) return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), __builtin_bit_cast(f16x2, 0u), acc, false);
  else return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, 0u), acc, false);
}

// Sums over the lanes up to and with this one, in 64 bits: within rows of 16 lanes, then the rows' last lanes to the rows behind.
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_from(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b)), CTRL, ROWS, 0xf, false));
  const uint32_t hi = uint32_t(__builtin_amdgcn_update_dpp(0, int(uint32_t(b >> 32)), CTRL, ROWS, 0xf, false));
  return x + __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}
__device__ __forceinline__ double scan64(double x) {
  x = add_from<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = add_from<0x112, 0xf>(x);
  x = add_from<0x114, 0xf>(x);
  x = add_from<0x118, 0xf>(x);
  x = add_from<0x142, 0xa>(x);  // row_bcast 15, to rows 1 and 3
  return add_from<0x143, 0xc>(x);  // row_bcast 31, to rows 2 and 3
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), lane)), hi = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b >> 32)), lane));
  return __builtin_bit_cast(double, uint64_t(hi) << 32 | lo);
}

// All wavefronts of the workgroup are here and their LDS accesses done. Loads from memory on their way stay there, for which __syncthreads
// would wait: the next chunk's rows.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The maximum over the wavefront, of numbers of 0 or more.
template <int CTRL, int ROWS>
__device__ __forceinline__ float max_from(float x) {
  return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float x) {
  x = max_from<0x111, 0xf>(x);
  x = max_from<0x112, 0xf>(x);
  x = max_from<0x114, 0xf>(x);
  x = max_from<0x118, 0xf>(x);
  x = max_from<0x142, 0xa>(x);
  x = max_from<0x143, 0xc>(x);
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

__device__ __forceinline__ float abs_max_halves(float x) { return fmaxf(x, __shfl_xor(x, 32)); }

// mfma_settle for several results at once.
__device__ __forceinline__ void settle(f32x16 (&x)[2]) { asm volatile("s_nop 15\n\ts_nop 15" : "+v"(x[0]), "+v"(x[1])); }
__device__ __forceinline__ void settle(f32x16 (&x)[4]) { asm volatile("s_nop 15\n\ts_nop 15" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3])); }

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
  float* const colf = reinterpret_cast<float*>(lds + L::kColF);
  float2* const since = reinterpret_cast<float2*>(lds + L::kSince);
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
    // Lane k: what the decays of the k segments between come to. (64 segments at a time; half a record is on its way while the one in
    // front of it joins.)
    constexpr int HT = KT / 2;
    f32x4 x[2][HT][4];
    auto load = [&](int k, int half) __attribute__((always_inline)) {
      const float* from = record(tile.part + tile.before - k) + half * (HT * 1024);
#pragma unroll
      for (int t = 0; t < HT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[half][t][i] = *reinterpret_cast<const f32x4*>(from + (t * 4 + i) * 256);
    };
    auto join = [&](float f, int half) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < HT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) S[half * HT + t][4 * i + e] = __builtin_fmaf(x[half][t][i][e], f, S[half * HT + t][4 * i + e]);
    };
    double front = 0.0;
    load(0, 0);
    for (int k0 = 0; k0 < tile.before; k0 += 64) {
      const int k = k0 + lane - 1;
      const double sums = front + scan64(k >= 0 && k < tile.before ? a.part_totals[size_t(tile.part + tile.before - k) * a.H + h] : 0.0);
      const int fs = __builtin_bit_cast(int, fast_exp2(float(sums)));
      front = lane_of(sums, 63);
#pragma unroll 1
      for (int i = 0; i < min(64, tile.before - k0); ++i) {
        const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(fs, i));
        load(k0 + i, 1);
        join(f, 0);
        load(min(k0 + i + 1, tile.before - 1), 0);
        join(f, 1);
      }
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
  const char *from_kq[NI], *from_v;  // the lane's first row of each piece in the next chunk
  uint32_t ld_kq[NI];
  uint32_t ld_v = uint32_t(2 * a.v_ld);
#pragma unroll
  for (int p = 0; p < NI; ++p) {
    const int it = tid + T * p;
    const bool isK = STATE || it < 2 * DK;  // (alike in a wavefront)
    const int b = (isK ? it : it - 2 * DK) % (2 * DK);
    ld_kq[p] = uint32_t(__builtin_amdgcn_readfirstlane(2 * (isK ? a.k_ld : a.q_ld)));
    from_kq[p] = reinterpret_cast<const char*>((isK ? a.K : a.Q) + size_t(kh) * DK) + (size_t(tile.row0) + 4 * piece_group<kParts>(b)) * ld_kq[p] + 16 * piece_part<kParts>(b);
  }
  from_v = reinterpret_cast<const char*>(a.V + dv0) + (size_t(tile.row0) + 4 * piece_group<vParts>(tid)) * ld_v + 16 * piece_part<vParts>(tid);
  // Row i of piece p (of NI: V's) of the next chunk; in the segment's last one rows behind the last are read as that one.
  auto fetch_row = [&](int p, int i) __attribute__((always_inline)) {
    if (p < NI) kq[p < NI ? p : 0][i] = *reinterpret_cast<const u32x4*>(from_kq[p < NI ? p : 0] + size_t(i) * ld_kq[p < NI ? p : 0]);
    else vv[i] = *reinterpret_cast<const u32x4*>(from_v + size_t(i) * ld_v);
  };
  // The n < 64 rows that start `ahead` rows behind the pointers' chunk.
  auto fetch_last = [&](int n, int ahead) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < NI; ++p) {
      const int r = 4 * piece_group<kParts>((tid + T * p) % (2 * DK));
#pragma unroll
      for (int i = 0; i < 4; ++i) kq[p][i] = *reinterpret_cast<const u32x4*>(from_kq[p] + int64_t(ahead + min(r + i, n - 1) - r) * int64_t(ld_kq[p]));
    }
    const int r = 4 * piece_group<vParts>(tid);
#pragma unroll
    for (int i = 0; i < 4; ++i) vv[i] = *reinterpret_cast<const u32x4*>(from_v + int64_t(ahead + min(r + i, n - 1) - r) * int64_t(ld_v));
  };
  auto fetch_decay = [&](int c) __attribute__((always_inline)) {  // (as it is: working on it here would be a wait)
    if (a.decay_ld) g_row = a.decay[(size_t(tile.row0) + min(64 * c + lane, tile.rows - 1)) * a.decay_ld + h];
  };
  auto fetch_on = [&](uint32_t rows) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < NI; ++p) from_kq[p] += size_t(rows) * ld_kq[p];
    from_v += size_t(rows) * ld_v;
  };
  auto fetch_all = [&](int c) __attribute__((always_inline)) {
    const int n = tile.rows - 64 * c;
    if (n >= 64) {
#pragma unroll
      for (int p = 0; p <= NI; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) fetch_row(p, i);
    } else {
      fetch_last(n, 0);
    }
    fetch_decay(c);
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

  if (n_chunks > 0) fetch_all(0);
  if (!STATE && tile.rows < 64) {  // no whole chunk that could be read again: the first row stands for it
#pragma unroll
    for (int p = 0; p < NI; ++p) {
      from_kq[p] -= size_t(4 * piece_group<kParts>((tid + T * p) % (2 * DK))) * ld_kq[p];
      ld_kq[p] = 0;
    }
    from_v -= size_t(4 * piece_group<vParts>(tid)) * ld_v;
    ld_v = 0;
  }
  double so_far = 0.0;
  for (int c = 0; c < n_chunks; ++c) {
    const int n = min(64, tile.rows - 64 * c);
    if (c > 0) lds_barrier();  // everybody is done with the chunk in front of this one
    if (n < 64) {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int it = tid + T * i;
        if (STATE || it < 2 * DK) clear_past(kq[i], 4 * piece_group<kParts>(it), n);
      }
      clear_past(vv, 4 * piece_group<vParts>(tid), n);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int it = tid + T * i;
      if (STATE && it >= 2 * DK) break;
      const bool isK = STATE || it < 2 * DK;
      const int b = isK ? it : it - 2 * DK;
      if (!STATE) put_rows(kq[i], isK ? L::kK : L::kQ, piece_group<kParts>(b), piece_part<kParts>(b));
      if (isK) put_columns(kq[i], L::kKT, piece_group<kParts>(b), piece_part<kParts>(b));
    }
    put_columns(vv, L::kVT, piece_group<vParts>(tid), piece_part<vParts>(tid));
    // What the chunk's decays come to. Of a head's own they are those of the chunk before, but for the first and the last.
    if (a.decay_ld || c == 0 || n < 64) {
      const double s = a.decay_ld ? scan64(lane < n ? double(decay_log2(g_row)) : 0.0) : double(g_const) * min(lane + 1, n);
      const double cl = lane_of(s, 63);
      so_far = STATE ? so_far + cl : 0.0;
      if (wave == 0) left[lane] = lane < n ? fast_exp2(float(cl - s)) : 0.0f;
      if (wave == NW - 1) {
        rowf[lane] = a.scale * fast_exp2(float(s));
        if (lane == 0) *total = fast_exp2(float(cl));
      }
      if (!STATE) {
#pragma unroll
        for (int i = 0; i < 4 / NW; ++i) {
          const int t = i ? 3 - wave : wave;
          const double b = t ? lane_of(s, 16 * t - 1) : 0.0;
          colf[64 * t + lane] = lane < 16 * t ? fast_exp2(float(b - s)) : 0.0f;
          const float hi = float(s - b);
          if (lane >> 4 == t) since[lane] = float2{hi, float(s - b - double(hi))};
        }
      }
    } else if (STATE) {
      so_far += double(g_const) * 64.0;
    }
    lds_barrier();
    if (STATE && c + 1 < n_chunks) {
      fetch_on(64);
      fetch_all(c + 1);
    }

    f32x16 O[2];
    float s_down = 1.0f;
    if constexpr (!STATE) {
      // P^T, 16 x 16 at a time: lane l has row 16 rt + l % 16 and columns 16 jt + 4 (l / 16) .. + 3. Every wavefront makes all four
      // tiles of its rows (the last one needs them all): without branches the rest can be laid under the next product.
      const int l16 = lane & 15, q4 = lane >> 4;
      int rt, row;
      f32x4 x[4];
      float row_scale, mx, p_up;
      f32x4 diagonal;
      auto make_p = [&](int which) __attribute__((always_inline)) {
        rt = which, row = 16 * rt + l16;
        const uint32_t q_at = place(L::kQ + row_part<DK>(row, q4)), k_at = place(L::kK + row_part<DK>(l16, q4));
        u32x4 qf[DK / 32];
#pragma unroll
        for (int kk = 0; kk < DK / 32; ++kk) qf[kk] = read(q_at ^ (kk << 6));
        // Weights: within the diagonal tile exp(c_i - c_j), left of it the product of what lies before and behind the tile's first row.
        const float2 ci = since[row];
        row_scale = a.scale * fast_exp2(ci.x + ci.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 cj = since[16 * rt + 4 * q4 + e];
          diagonal[e] = a.scale * fast_exp2((ci.x - cj.x) + (ci.y - cj.y));
        }
        mx = 0.0f;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) x[jt] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < DK / 32; ++kk)
#pragma unroll
          for (int jt = 0; jt < 4; ++jt) x[jt] = mfma16x32<DT>(read((k_at ^ (kk << 6)) + jt * (32 * DK)), qf[kk], x[jt]);
      };
      auto weigh_p = [&](int jt) __attribute__((always_inline)) {
        const f32x4 before = *reinterpret_cast<const f32x4*>(colf + 64 * rt + 16 * jt + 4 * q4);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = x[jt][e] * (jt == rt ? diagonal[e] : row_scale * before[e]);
          asm("" : "+v"(y));  // (left alone the compiler branches around the work of each masked weight)
          x[jt][e] = 16 * jt + 4 * q4 + e <= row ? y : 0.0f;
          mx = fmaxf(mx, fabsf(x[jt][e]));
        }
      };
      auto scale_p = [&]() __attribute__((always_inline)) {
        if constexpr (DT == ESP_F16) {
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          float down;
          scale_for(mx, kOutputScale, p_up, down);
          pinv[row] = down;  // (four lanes with the same)
        }
      };
      auto put_p = [&](int jt) __attribute__((always_inline)) {
        if constexpr (DT == ESP_F16) x[jt] *= p_up;
        uint32_t w0 = pack2<DT>(x[jt][0], x[jt][1]), w1 = pack2<DT>(x[jt][2], x[jt][3]);
        asm("" : "+v"(w0), "+v"(w1));
        const uint32_t r0 = pack2<DT>(x[jt][0] - unpack_lo<DT>(w0), x[jt][1] - unpack_hi<DT>(w0));
        const uint32_t r1 = pack2<DT>(x[jt][2] - unpack_lo<DT>(w1), x[jt][3] - unpack_hi<DT>(w1));
        // Rows 0 .. 31 have no place for columns 32 .. 63, all of them zeros.
        const bool real = jt <= (rt | 1);
        const uint32_t to = base + uint32_t(real ? L::kP + p_part(row, 2 * jt + (q4 >> 1)) + 8 * (q4 & 1) : L::kNone + 8 * lane);
        *reinterpret_cast<lds_u32x2_out*>(to) = u32x2{w0, w1};
        *reinterpret_cast<lds_u32x2_out*>(to + (real ? kPBytes : 0)) = u32x2{r0, r1};
      };
      if constexpr (NW == 2) {
        make_p(3 - wave);
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) weigh_p(jt);
        scale_p();
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) put_p(jt);
      }
      make_p(wave);
      // (Q S)^T, a step of 16 dims at a time; the next step's part of S is split, and P's weights are worked out, under the products.
      O[0] = f32x16{};
      O[1] = f32x16{};
      float s_up = 1.0f;
      if constexpr (DT == ESP_F16) {
        float sx = 0.0f;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int e = 0; e < 16; ++e) sx = fmaxf(sx, fabsf(S[t][e]));
        if (__builtin_expect(__any(sx == INFINITY), 0)) {  // infinities are not what the others are scaled by
          sx = 0.0f;
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) sx = fabsf(S[t][e]) < INFINITY ? fmaxf(sx, fabsf(S[t][e])) : sx;
        }
        sx = wave_max(sx);
        scale_for(sx, kOutputScale, s_up, s_down);
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) mfma_settle(x[jt]);
      }
      const uint32_t q_at = place(L::kQ + row_part<DK>(l32, hb));
      constexpr int NS = DK / 16, PER = 8 / NS;  // steps; of the eight pieces of P's work how many go with each
      u32x4 sp[2][2], q[2][2];
      auto step_in = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) q[ks & 1][r] = read((q_at ^ (ks << 5)) + r * (64 * DK));
      };
      auto step_split = [&](int ks) __attribute__((always_inline)) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = S[ks >> 1][8 * (ks & 1) + e];
        split8<DT, 2>(y, s_up, sp[ks & 1]);
      };
      // The next chunk's rows are asked for here, a few a step: all at once they stand in line for a quarter of the chunk's time. Without
      // another whole chunk it is the last whole one's rows once more, and the rest of the segment's are asked for behind.
      const bool next_whole = tile.rows - 64 * (c + 1) >= 64;
      fetch_on(next_whole ? 64 : 0);
      constexpr int LOADS = 4 * (NI + 1), LPS = (LOADS + NS - 1) / NS;
      step_in(0);
      step_split(0);
#pragma unroll
      for (int ks = 0; ks < NS; ++ks) {
        if (ks + 1 < NS) step_in(ks + 1);
#pragma unroll
        for (int y = ks * LPS; y < (ks + 1) * LPS && y < LOADS; ++y) fetch_row(y >> 2, y & 3);
#pragma unroll
        for (int v = 0; v < 2; ++v)
#pragma unroll
          for (int r = 0; r < 2; ++r) O[r] = mfma32x16<DT>(sp[ks & 1][v], q[ks & 1][r], O[r]);
        if (ks + 1 < NS) step_split(ks + 1);
#pragma unroll
        for (int y = ks * PER; y < (ks + 1) * PER; ++y) {
          if (y < 4) weigh_p(y);
          if (y == 3) scale_p();
          if (y >= 4) put_p(y - 4);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 16, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (c + 1 < n_chunks && !next_whole) {
        fetch_last(tile.rows - 64 * (c + 1), 64);
      }
      if (c + 1 < n_chunks) fetch_decay(c + 1);
      lds_barrier();  // P is there, and nobody reads Q and K any more
    }
    // Rows of O leave through LDS, where Q and K were, a wavefront's 64 rows of 64 bytes each, 16-byte parts turned by the row; written behind
    // the products, read and stored under those of the state.
    auto row_at = [&](int r, int p) { return lds + L::kQ + wave * 4096 + r * 64 + ((p ^ ((r >> 2) & 3)) << 4); };
    u32x4 rows_out[4];
    auto read_rows = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 4 && !STATE; ++i) rows_out[i] = *reinterpret_cast<const u32x4*>(row_at(16 * i + (lane >> 2), lane & 3));
    };
    auto store_rows = [&]() __attribute__((always_inline)) {
      char* const to = reinterpret_cast<char*>(a.O + (size_t(tile.row0) + 64 * size_t(c)) * a.o_ld + dv0 + 32 * wave) +
                       uint32_t(lane >> 2) * uint32_t(2 * a.o_ld) + 16 * (lane & 3);
#pragma unroll
      for (int i = 0; i < 4 && !STATE; ++i)
        if (16 * i + (lane >> 2) < n) *reinterpret_cast<u32x4*>(to + i * (32 * size_t(a.o_ld))) = rows_out[i];
    };
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
        for (int e = 0; e < 4; ++e) nf = times_zero2<DT>(vr[ks][e], nf);
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
      const uint32_t p_at[2] = {place(L::kP + p_part(l32, hb)), place(L::kP + p_part(32 + l32, hb))};
      u32x4 pq[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) pq[i] = read(p_at[i & 1] + (i >> 1) * kPBytes);
      settle(O);
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        float f = rowf[32 * rt + l32];
        if constexpr (DT == ESP_F16) {
          f *= s_down;
          O[rt] *= f;
          O[rt] *= 1.0f / pinv[32 * rt + l32];  // (a power of two)
        } else {
          O[rt] *= f;
        }
      }
      // Twelve products: of both halves of the rows in turn as long as there are two.
      auto which = [](int i) { return i < 8 ? i >> 2 : 2 + ((i - 8) >> 1); };   // 16 columns
      auto of_rows = [](int i) { return i < 8 ? i & 1 : 1; };
      auto p_in = [&](int i) {
        const int v = i < 8 ? (i >> 1) & 1 : i & 1;
        return read((p_at[of_rows(i)] ^ (which(i) << 5)) + v * kPBytes);
      };
#pragma unroll
      for (int i = 0; i < 12; ++i) {
        if (i % 4 == 0 && i < 8) {
#pragma unroll
          for (int y = i + 4; y < i + 8; ++y) pq[y & 7] = p_in(y);
        }
        O[of_rows(i)] = mfma32x16<DT>(vr[which(i)], pq[i & 7], O[of_rows(i)]);
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
      settle(O);
#pragma unroll
      for (int rt = 0; rt < 2; ++rt) {
        const int row = 32 * rt + l32;
        if (__builtin_expect(odd, 0)) {
          // Rows 8 (e / 4) + 4 hb + e % 4 of the wavefront's part of V^T: their turns differ by constants.
#pragma unroll 1
          for (int j = 0; j <= row; ++j) {
            const float p = unpack_lo<DT>(*reinterpret_cast<const uint16_t*>(lds + L::kP + p_part(row, j >> 3) + 2 * (j & 7)));
            const uint32_t at = place(L::kVT + (32 * wave + 4 * hb) * 128 + (((j >> 3) ^ (2 * hb) ^ (2 * (wave & 1))) << 4) + 2 * (j & 7));
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              constexpr auto turn = [](int d) { return ((d >> 1) & 7) ^ ((d >> 4) & 1); };
              const int d = 8 * (e >> 2) + (e & 3);
              const float v = unpack_lo<DT>(*reinterpret_cast<const __attribute__((address_space(3))) uint16_t*>((at ^ (turn(d) << 4)) + d * 128));
              if (!(fabsf(v) < INFINITY)) O[rt][e] += p * v;
            }
          }
        }
        if constexpr (DT == ESP_F16) O[rt] *= pinv[row];
      }
      if (__builtin_expect(odd, 0)) read_v();
#pragma unroll
      for (int rt = 0; rt < 2; ++rt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<u32x2*>(row_at(32 * rt + l32, i) + 8 * hb) =
              u32x2{pack2<DT>(O[rt][4 * i], O[rt][4 * i + 1]), pack2<DT>(O[rt][4 * i + 2], O[rt][4 * i + 3])};
      __builtin_amdgcn_wave_barrier();
      asm volatile("" ::: "memory");
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
          split8<DT, NV>(x, up, vs[ks]);
        }
        f32x16 d[2];
        auto product = [&](int t) __attribute__((always_inline)) {
          d[t & 1] = f32x16{};
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const u32x4 k = read((k_at ^ ((ks ^ (t & 1)) << 5)) + t * 4096);
#pragma unroll
            for (int v = 0; v < NV; ++v) d[t & 1] = mfma32x16<DT>(k, vs[ks][v], d[t & 1]);
          }
        };
        read_rows();
        product(0);
        store_rows();
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          if (t + 1 < KT) product(t + 1);
          mfma_settle(d[t & 1]);
#pragma unroll
          for (int e = 0; e < 16; ++e) S[t][e] = __builtin_fmaf(d[t & 1][e], down, S[t][e] * f);
        }
      } else {
#pragma unroll
        for (int t = 0; t < KT; ++t) S[t] *= f;
        // The next 16 rows' values are weighed and split under the products of these.
        u32x4 vs[2][NV], k[2][KT];
        auto step_in = [&](int ks) __attribute__((always_inline)) {
#pragma unroll
          for (int t = 0; t < KT; ++t) k[ks & 1][t] = read((k_at ^ ((ks ^ (t & 1)) << 5)) + t * 4096);
        };
        auto step_split = [&](int ks) __attribute__((always_inline)) {
          float x[8];
          weighted(ks, x);
          split8<DT, NV>(x, 1.0f, vs[ks & 1]);
        };
        step_in(0);
        step_split(0);
        read_rows();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          if (ks < 3) step_in(ks + 1);
#pragma unroll
          for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int t = 0; t < KT; ++t) S[t] = mfma32x16<DT>(k[ks & 1][t], vs[ks & 1][v], S[t]);
          if (ks < 3) step_split(ks + 1);
#pragma unroll
          for (int y = 0; y < NV * KT; ++y) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 84 / (NV * KT), 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          if (ks == 0) store_rows();
        }
        settle(S);
      }
    } else {
      read_rows();
      store_rows();
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

// As many columns a workgroup as leave two workgroups for every compute unit. 32 heads of 128 x 128, bf16, of 128, 64 and 32 columns: 4 sequences
// of 5 rows 7.8, 7.3 and 6.8 us; 8 of 5 rows 9.5, 9.0 and 10.1; 32 of one row 21.2, 22.4 and 23.8.
template <int DT, int DK>
hipError_t launch_few(const LinearArgs& a, int n, hipStream_t st) {
  if (a.dv % 128 == 0 && long(a.H) * (a.dv / 128) * n >= 2 * kComputeUnits) return launch_few_t<DT, 128, DK>(a, n, st);
  if (long(a.H) * (a.dv / 64) * n >= 2 * kComputeUnits) return launch_few_t<DT, 64, DK>(a, n, st);
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
