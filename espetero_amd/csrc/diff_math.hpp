// What the differential attention kernels share: their argument block, the key range of a tile, and how a pair's two
// accumulators become an output row.
#pragma once

#include "common.hpp"

namespace esp {

constexpr int kDiffHD = 128;             // dims of a query or key head
constexpr int kDiffVD = 2 * kDiffHD;     // dims of a pair's values and output

// Everything a differential attention kernel reads, passed by value.
struct DiffArgs {
  const uint16_t* Q;
  const uint16_t* pool;
  const int32_t* blocks;
  uint16_t* O;
  const esp_tile* tiles;
  const esp_tree* trees;
  float* parts_o;   // [part][KV pair][map][cols][256]  unnormalised
  float* parts_ml;  // [part][KV pair][map][cols][2]    running max (log2 units), sum
  const float* weight;  // [query pair]
  const float* norm_w;  // [256], or null: no norm
  int32_t H, Hkv, G, q_ld, bt, window, ring, R, cols;  // G: query pairs per KV pair
  float scale_log2, eps, factor;
  uint64_t kv_base;
};

// Pool element where (block, KV head) starts.
__device__ __forceinline__ size_t diff_head_base(const DiffArgs& a, int b, int kvh) {
  return size_t(a.kv_base) + (size_t(b) * size_t(a.Hkv) + size_t(kvh)) * size_t(2 * a.bt * kDiffHD);
}
// The pool's block behind a tree's block number bi: from its list, or in its slot's ring.
__device__ __forceinline__ int diff_block(const DiffArgs& a, int table, int bi) {
  using const_i32 = const int32_t __attribute__((address_space(4)));  // read only: scalar loads
  return a.ring ? table + bi % a.ring : ((const_i32*)a.blocks)[table + bi];
}

// The keys a tile scans, [lo, hi) in cache positions: its cached range and, on a `last` tile, the rows of the pass behind it, which
// lie in the pool at positions P + row. Both at once only where they meet: the cached range then ends at P and b0 is 0.
struct DiffRange {
  int lo, hi, rr0, rows;  // rr0: the tile's first row within its tree; rows: live ones
};
__device__ __forceinline__ DiffRange diff_range(const esp_tile& t, const esp_tree& tr, int R, int window) {
  DiffRange d;
  d.rr0 = t.r0 - tr.base;
  d.rows = min(R, tr.M - d.rr0);
  const int k1 = min(t.k1, tr.P);  // INT32_MAX: up to the tree's cached length as it is now
  d.lo = t.k0;
  d.hi = k1;
  if (t.last) {
    int e = d.rr0 + d.rows;  // one past the last row any row of the tile sees
    if (t.last >= 2) e = min(e, t.last - 1);
    if (k1 <= t.k0) d.lo = tr.P + t.b0;
    d.hi = tr.P + e;
  }
  if (window > 0) d.lo = max(d.lo, tr.P + d.rr0 - window + 1);  // what no row of the tile sees any more
  d.hi = max(d.hi, d.lo);
  return d;
}

// 0 for a row that has seen no key; NaN stays NaN.
__device__ __forceinline__ float diff_inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }

// A wavefront's 256 dims of one (row, pair), 4 per lane: o1 and o2 unnormalised with sums l1 and l2. The difference of the two maps'
// outputs, its norm over the pair's dims and the factor in fp32, then the one rounding to the storage type.
template <int DT>
__device__ __forceinline__ void diff_finish(const DiffArgs& a, int row, int pair, int lane, f32x4 o1, float l1, f32x4 o2, float l2) {
  const float i1 = diff_inverse(l1), i2 = diff_inverse(l2) * a.weight[pair];
  f32x4 o = o1 * i1 - o2 * i2;
  float f = a.factor;
  if (a.norm_w) {
    float ss = o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3];
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) ss += __shfl_xor(ss, x);
    f *= rsqrtf(ss * (1.0f / kDiffVD) + a.eps);
    o *= *reinterpret_cast<const f32x4*>(a.norm_w + 4 * lane);
  }
  o *= f;
  *reinterpret_cast<u32x2*>(a.O + size_t(row) * a.q_ld + size_t(pair) * kDiffVD + 4 * lane) = u32x2{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
}

// Infinities and NaN among the two storage elements of a dword, as a mask of the elements' bits.
template <int DT>
__device__ __forceinline__ uint32_t not_finite2(uint32_t w) {
  constexpr uint32_t e = DT == ESP_F16 ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0xffffu : 0u) | ((w >> 16 & e) == e ? 0xffff0000u : 0u);
}

// 1.0 in the storage type where an element is an infinity of the given sign or NaN, else 0. A product of such marks with the weights is
// finite whatever they are, and positive where a row sees such a value.
template <int DT>
__device__ __forceinline__ uint32_t not_finite_marks(uint32_t w, bool negative) {
  constexpr uint32_t e = DT == ESP_F16 ? 0x7c00u : 0x7f80u, one = DT == ESP_F16 ? 0x3c00u : 0x3f80u;
  auto mark = [&](uint32_t x) { return (x & e) == e && ((x & 0x7fffu) != e || (x >> 15 != 0) == negative) ? one : 0u; };
  return mark(w & 0xffffu) | mark(w >> 16) << 16;
}

}  // namespace esp
