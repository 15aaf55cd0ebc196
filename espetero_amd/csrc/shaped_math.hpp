// What the kernels of attention with shaped scores share: their argument block, what a row sees, how a product becomes a score, and
// which keys a tile scans.
#pragma once

#include "common.hpp"
#include "diff_math.hpp"

namespace esp {

// Everything a kernel of attention with shaped scores reads, passed by value.
struct ShapedArgs {
  const uint16_t* Q;
  const uint16_t* pool;
  const int32_t* blocks;
  uint16_t* O;
  const esp_tile* tiles;
  const esp_tree* trees;
  float* parts_o;   // [part][Hkv][cols][head_dim]  unnormalised
  float* parts_ml;  // [part][Hkv][cols][2]         running max (log2 units), sum
  const float* slopes;  // [H], or null
  const int2* spans;    // [n_rows] (first key, end of what is seen whichever way round), or null
  int32_t H, Hkv, G, q_ld, bt, window, ring, R, cols;
  float scale_log2;  // without a cap: scale in log2 units; with one: 2 scale log2(e) / cap
  float cap_log2;    // cap in log2 units
  // cap tanh(scale q.k / cap) in log2 units as q.k times a polynomial of (q.k)^2, for |q.k| < tanh_below. tanh(z) / z fitted in z^2 for
  // |z| < 0.7: six steps of 2^-24 of tanh off in fp32. 0, or fewer terms and a nearer bound, where fp32 does not hold the coefficients.
  float tanh_c[5], tanh_below;
  float tanh_s[3], tanh_short;  // likewise for |z| < 0.2, where three terms do
  uint64_t kv_base;
};

__device__ __forceinline__ int shaped_block(const ShapedArgs& a, int table, int bi) {
  using const_i32 = const int32_t __attribute__((address_space(4)));  // read only: scalar loads
  return a.ring ? table + bi % a.ring : ((const_i32*)a.blocks)[table + bi];
}

// The keys [from, end) that a row at position q sees of a tree with n_keys.
struct Sight {
  int from, end;
};
__device__ __forceinline__ Sight shaped_sight(const ShapedArgs& a, int row, int q, int n_keys) {
  Sight s{0, q + 1};
  if (a.spans) {
    const int2 span = a.spans[row];
    s.end = min(max(q + 1, span.y), n_keys);
    s.from = min(max(span.x, 0), s.end);  // (a row that sees nothing: no number that later sums could carry past 32 bits)
  }
  if (a.window > 0) s.from = max(s.from, q - a.window + 1);
  return s;
}

// x = scale q.k through the cap, in log2 units. cap tanh(x / cap) = cap (1 - 2 / (exp(2 x / cap) + 1)) holds for infinite x too, but is off by as
// many steps of the cap as of x: small x go through the polynomial.
__device__ __forceinline__ float shaped_tanh_low(const ShapedArgs& a, float dot, float add) {
  const float u = dot * dot;
  float p = __builtin_fmaf(u, a.tanh_c[4], a.tanh_c[3]);
  p = __builtin_fmaf(u, p, a.tanh_c[2]);
  p = __builtin_fmaf(u, p, a.tanh_c[1]);
  p = __builtin_fmaf(u, p, a.tanh_c[0]);
  return __builtin_fmaf(dot, p, add);
}
__device__ __forceinline__ float shaped_tanh_short(const ShapedArgs& a, float dot, float add) {
  const float u = dot * dot;
  return __builtin_fmaf(dot, __builtin_fmaf(u, __builtin_fmaf(u, a.tanh_s[2], a.tanh_s[1]), a.tanh_s[0]), add);
}
__device__ __forceinline__ float shaped_tanh_high(const ShapedArgs& a, float dot, float add) {
  return __builtin_fmaf(-2.0f * a.cap_log2, __builtin_amdgcn_rcpf(fast_exp2(dot * a.scale_log2) + 1.0f), a.cap_log2 + add);
}
template <bool CAP>
__device__ __forceinline__ float shaped_score(const ShapedArgs& a, float dot) {
  if constexpr (!CAP) return dot * a.scale_log2;
  const float high = shaped_tanh_high(a, dot, 0.0f), low = shaped_tanh_low(a, dot, 0.0f);
  return fabsf(dot) < a.tanh_below ? low : high;
}

// The keys a tile scans, [lo, hi) in cache positions, of those that its rows see at all, [from, end): its cached range and, on a `last` tile,
// the rows of the pass behind it, which lie in the pool at positions P + row - up to `end` where the tile's range of them is open. Both at once
// only where they meet.
__device__ __forceinline__ Sight shaped_range(const esp_tile& t, const esp_tree& tr, int from, int end) {
  const int k1 = min(t.k1, tr.P);  // INT32_MAX: up to the tree's cached length as it is now
  Sight d{t.k0, k1};
  if (t.last) {
    if (k1 <= t.k0) d.from = tr.P + t.b0;
    d.end = t.last >= 2 ? tr.P + t.last - 1 : INT32_MAX;
  }
  d.from = max(d.from, from);
  d.end = max(min(d.end, end), d.from);
  return d;
}

// What sums taken from reference m count for beside a reference M of m or more; m is -inf where no key has been seen. Never zero for keys that
// have: a sum may hold an infinite value, which is no less infinite for weighing next to nothing (2^-126 of finite ones is lost in any output).
__device__ __forceinline__ float shaped_share(float m, float M) { return m == -INFINITY ? 0.0f : fmaxf(fast_exp2(m - M), 0x1p-126f); }

__device__ __forceinline__ float shaped_inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }  // 0: a row that has seen no key; NaN stays

}  // namespace esp
