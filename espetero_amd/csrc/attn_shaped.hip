// Attention over the paged pool with shaped scores: a row at position p weighs a key at position j by the softmax of
//   x = scale q.k ;  x = cap tanh(x / cap) with a cap ;  x -= slope[h] |p - j| with slopes
// over the keys it sees: those of its span, up to its own or to the span's end, the last `window` of them on a sliding layer.
//
// Streaming kernel: decode and short trees. Bound by HBM: every visible key's K and V are read once for all G query heads of a KV head and
// all rows of the tile. One workgroup is one tile and one KV head; up to 16 packed rows (row in tile * G + head of the group) are the columns
// of a matrix tile, NC such tiles. A wavefront takes 16-key units round robin straight from HBM with the next unit's loads in
// flight; the four wavefronts' sums meet in LDS at the end. 24 sequences of 300 to 9000 keys, 32 / 8 heads of 128 dims: 90 us for 540 MB, 6.0 TB/s
// of the 6.6 that a plain read of such pages reaches, and 5 us for the merge; two or three units ahead in place of one: 1 us less.
#include "shaped_math.hpp"

namespace esp {

namespace {

template <int HD>
struct ShapedUnit {  // 16 keys: K and V^T
  u32x4 k[HD / 32];  // [32-dim group]: key = lane % 16, dims 32 kk + 8 (lane / 16) ..
  u32x2 v[HD / 16];  // [16-dim group]: dim = 16 mt + lane % 16, keys 4 (lane / 16) ..
};

}  // namespace

template <int DT, int HD, int NC, bool CAP>
__global__ __launch_bounds__(256, HD == 128 && NC == 1 ? 2 : 1) void attn_shaped_stream_kernel(const ShapedArgs a) {
  constexpr int MT = HD / 16, KK = HD / 32, LDO = HD + 4, VEC = HD / 64;
  extern __shared__ float smem[];  // [4 wavefronts][NC * 16 columns][LDO] O, then [4][NC * 16][2] m, l
  const int kvh = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, q4 = lane >> 4;
  const esp_tile tile = a.tiles[blockIdx.y];
  const esp_tree tree = a.trees[tile.tree];
  const int table = tile.pad > 0 ? tile.pad - 1 : tree.table;
  const int rr0 = tile.r0 - tree.base, rows = min(a.R, tree.M - rr0), cols_live = rows * a.G;

  // ---- this lane's packed rows: Q operands, what they see, their slopes
  u32x4 qf[NC][KK];
  int qpos[NC];
  Sight sight[NC];
  float slope[NC];
  int some_from = INT32_MAX, some_end = 0, all_from = 0, all_end = INT32_MAX;  // over the tile's rows
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = 16 * c + c16;
    const bool ok = col < cols_live;
    const int m = ok ? col / a.G : 0, hg = ok ? col - m * a.G : 0;
    qpos[c] = tree.P + rr0 + m;
    const uint16_t* qp = a.Q + size_t(tile.r0 + m) * a.q_ld + size_t(kvh * a.G + hg) * HD + 8 * q4;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qf[c][kk] = ok ? *reinterpret_cast<const u32x4*>(qp + 32 * kk) : u32x4{0, 0, 0, 0};
    slope[c] = a.slopes ? a.slopes[kvh * a.G + hg] * kLog2e : 0.0f;
    sight[c] = shaped_sight(a, tile.r0 + m, qpos[c], tree.P + tree.M);
    some_from = min(some_from, sight[c].from);
    some_end = max(some_end, sight[c].end);
    all_from = max(all_from, sight[c].from);
    all_end = min(all_end, sight[c].end);
  }
  if (rows > 1) {  // (columns without a row have the first one's)
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) {
      some_from = min(some_from, __shfl_xor(some_from, x));
      some_end = max(some_end, __shfl_xor(some_end, x));
      all_from = max(all_from, __shfl_xor(all_from, x));
      all_end = min(all_end, __shfl_xor(all_end, x));
    }
  }
  some_from = __builtin_amdgcn_readfirstlane(some_from), some_end = __builtin_amdgcn_readfirstlane(some_end);
  all_from = __builtin_amdgcn_readfirstlane(all_from), all_end = __builtin_amdgcn_readfirstlane(all_end);
  const Sight rg = shaped_range(tile, tree, some_from, some_end);

  // ---- 16-key units; interior ones are seen whole by every row of the tile
  const int u_lo = rg.from >> 4, u_hi = (rg.end + 15) >> 4;
  const int n_units = rg.end > rg.from ? u_hi - u_lo : 0;
  int ui0 = u_lo, ui1 = u_lo;
  if (n_units) {
    ui0 = min((max(rg.from, all_from) + 15) >> 4, u_hi);
    ui1 = max(ui0, min(rg.end, all_end) >> 4);
  }

  f32x4 acc[NC][MT];
  float m_run[NC], l_run[NC];

  const uint32_t lane_k = uint32_t(c16 * HD + 8 * q4) * 2, lane_v = uint32_t(c16 * kVtDim + 4 * q4) * 2;
  const uint32_t head = uint32_t(2 * a.bt * HD) * 2, to_v = uint32_t(a.bt * HD) * 2;  // bytes of one (block, KV head); from its K to its V^T
  const uint64_t block_bytes = uint64_t(a.Hkv) * head;
  const char* const pool = reinterpret_cast<const char*>(a.pool + a.kv_base) + uint64_t(kvh) * head;
  auto block_of = [&](int u) {  // (a sub-block of V^T starts as far behind the first as its first token's K row does)
    const int key = u << 4, bi = key / a.bt;
    return pool + uint64_t(uint32_t(shaped_block(a, table, bi))) * block_bytes + uint32_t(key - bi * a.bt) * (HD * 2);
  };
  auto load = [&](int u, ShapedUnit<HD>& U) {
    const char* const kp = block_of(u);
    const char* const vp = kp + to_v;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) U.k[kk] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + lane_k + 64 * kk));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) U.v[mt] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vp + lane_v + 32 * kVtDim * mt));
  };
  auto scores = [&](int u, const ShapedUnit<HD>& U, f32x4 (&s)[NC]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      s[c] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) s[c] = mfma16x32<DT>(U.k[kk], qf[c][kk], s[c]);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      mfma_settle(s[c]);
      const float ago = float((u << 4) + 4 * q4 - qpos[c]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[c][e] = shaped_score<CAP>(a, s[c][e]) - slope[c] * fabsf(ago + float(e));
    }
  };
  // Online softmax over scores x (log2 units, -inf where masked), then O^T += V^T . P^T. The matrix product takes P in the storage type, as
  // the sum of two such numbers, 16 bits or more: one alone makes the output 1.4 times as inexact as its own rounding does, and the
  // second product waits for memory anyway. Of fp16 the largest weight is 2^15, so that a number's last step, 2^-24, is 2^-39 of it.
  auto softmax_pv = [&](const ShapedUnit<HD>& U, const f32x4 (&x)[NC]) {
    bool any_change = false;
    f32x4 p[NC];
    float corr[NC];
    u32x2 pb[NC], pl[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = fmaxf(fmaxf(x[c][0], x[c][1]), fmaxf(x[c][2], x[c][3]));
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m_run[c], mx);
      const float m_safe = (m_new == -INFINITY) ? 0.0f : m_new;
      corr[c] = fmaxf(fast_exp2(m_run[c] - m_safe), 0x1p-126f);  // (what is infinite stays so)
      any_change = any_change || (m_new > m_run[c]);
      m_run[c] = m_new;
#pragma unroll
      for (int e = 0; e < 4; ++e) p[c][e] = fast_exp2(DT == ESP_F16 ? (x[c][e] - m_safe) + 15.0f : x[c][e] - m_safe);
      pb[c] = u32x2{pack2<DT>(p[c][0], p[c][1]), pack2<DT>(p[c][2], p[c][3])};
      pl[c] = u32x2{pack2<DT>(p[c][0] - unpack_lo<DT>(pb[c].x), p[c][1] - unpack_hi<DT>(pb[c].x)),
                    pack2<DT>(p[c][2] - unpack_lo<DT>(pb[c].y), p[c][3] - unpack_hi<DT>(pb[c].y))};
      l_run[c] = l_run[c] * corr[c] + sum2<DT>(pl[c].x, sum2<DT>(pb[c].x, sum2<DT>(pl[c].y, sum2<DT>(pb[c].y, 0.0f))));  // (as the product takes them)
    }
    if (__any(any_change)) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) acc[c][mt] *= corr[c];
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        acc[c][mt] = mfma16x16<DT>(U.v[mt], pb[c], acc[c][mt]);
        acc[c][mt] = mfma16x16<DT>(U.v[mt], pl[c], acc[c][mt]);
      }
  };
  auto interior = [&](int u, const ShapedUnit<HD>& U) {
    f32x4 s[NC];
    scores(u, U, s);
    softmax_pv(U, s);
  };
  // A unit with keys that some row does not see, or (careful) with values that may be infinite.
  auto edge = [&](int u, ShapedUnit<HD>& U, bool careful) {
    // Keys outside the range may be memory never written: their V must not reach the products (0 * NaN).
    const int jv = (u << 4) + 4 * q4;
    uint32_t in[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) in[e] = (jv + e >= rg.from && jv + e < rg.end) ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
    uint32_t bad = 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      U.v[mt].x &= in[0] | in[1];
      U.v[mt].y &= in[2] | in[3];
      bad |= not_finite2<DT>(U.v[mt].x) | not_finite2<DT>(U.v[mt].y);
    }
    // Nor may the infinite V of a key that one row sees reach a row that does not, or meet a weight's second number, which may be zero or below:
    // such elements leave the product, and a product of marks in their places says which rows see them.
    const bool rare = (rows > 1 || careful) && __any(bad != 0);
    if (rare) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        U.v[mt].x &= ~not_finite2<DT>(U.v[mt].x);
        U.v[mt].y &= ~not_finite2<DT>(U.v[mt].y);
      }
    }
    f32x4 s[NC];
    scores(u, U, s);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int from = max(rg.from, sight[c].from), n = max(0, min(rg.end, sight[c].end) - from);
        s[c][e] = uint32_t(jv + e - from) < uint32_t(n) ? s[c][e] : -INFINITY;
      }
    softmax_pv(U, s);
    if (__builtin_expect(rare, 0)) {
      constexpr uint32_t one = DT == ESP_F16 ? 0x3c00u : 0x3f80u;
      u32x2 sees[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int from = max(rg.from, sight[c].from), n = max(0, min(rg.end, sight[c].end) - from);
        auto seen = [&](int e) { return uint32_t(jv + e - from) < uint32_t(n) ? one : 0u; };
        sees[c] = u32x2{seen(0) | seen(1) << 16, seen(2) | seen(3) << 16};
      }
      const char* const vp = block_of(u) + to_v + lane_v;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(vp + 32 * kVtDim * mt);
        const uint32_t lo = v.x & (in[0] | in[1]), hi = v.y & (in[2] | in[3]);
#pragma unroll
        for (int neg = 0; neg < 2; ++neg)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            f32x4 seen = mfma16x16<DT>(u32x2{not_finite_marks<DT>(lo, neg != 0), not_finite_marks<DT>(hi, neg != 0)}, sees[c], f32x4{0, 0, 0, 0});
            mfma_settle(seen);
            mfma_settle(acc[c][mt]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (seen[e] > 0.0f) acc[c][mt][e] += neg ? -INFINITY : INFINITY;
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };

  auto clear = [&] {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      m_run[c] = -INFINITY;
      l_run[c] = 0.0f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) acc[c][mt] = f32x4{0, 0, 0, 0};
    }
  };
  auto odd = [&] {  // is some sum infinite or NaN?
    float nf = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        mfma_settle(acc[c][mt]);
#pragma unroll
        for (int e = 0; e < 4; ++e) nf = __builtin_fmaf(acc[c][mt][e], 0.0f, nf);
      }
    return __any(nf != 0.0f) != 0;  // (NaN, or 0)
  };
  const int n_int = ui1 - ui0, n_lo = ui0 - u_lo, n_edge = n_units - n_int;
  const int n_mine = n_int > wave ? (n_int - wave + 3) / 4 : 0;
  const int u0 = ui0 + wave, e0 = (wave + 4 - n_int % 4) % 4;  // edges go on with the round robin
  auto edge_unit = [&](int i) { return i < n_lo ? u_lo + i : ui1 + (i - n_lo); };
  ShapedUnit<HD> U[2];
  clear();
  if (n_mine > 0) {
    load(u0, U[0]);
    int i = 0;
    for (; i + 2 < n_mine; i += 2) {
      load(u0 + 4 * (i + 1), U[1]);
      interior(u0 + 4 * i, U[0]);
      load(u0 + 4 * (i + 2), U[0]);
      interior(u0 + 4 * (i + 1), U[1]);
    }
    if (i + 2 == n_mine) {
      load(u0 + 4 * (i + 1), U[1]);
      interior(u0 + 4 * i, U[0]);
      interior(u0 + 4 * (i + 1), U[1]);
    } else {
      interior(u0 + 4 * i, U[0]);
    }
  }
  for (int i = e0; i < n_edge; i += 4) {
    load(edge_unit(i), U[0]);
    edge(edge_unit(i), U[0], false);
  }
  // Infinite and NaN values of an interior unit go into its products as they are, where a weight's second number, or one that has vanished, makes
  // NaN of an infinity: a wavefront that has met one takes its units once more, in the same order, each with such values taken out.
  if (__builtin_expect(odd(), 0)) {
    clear();
#pragma unroll 1
    for (int i = e0 - 4 * n_mine; i < n_edge; i += 4) {
      const int u = i < e0 ? u0 + i - e0 + 4 * n_mine : edge_unit(i);
      load(u, U[0]);
      edge(u, U[0], true);
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) mfma_settle(acc[c][mt]);
  }

  // ---- merge the 4 wavefronts in order
  float* o_sh = smem;
  float* ml_sh = smem + 4 * NC * 16 * LDO;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = 16 * c + c16;
    float l = l_run[c];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (q4 == 0) {
      ml_sh[(wave * NC * 16 + col) * 2] = m_run[c];
      ml_sh[(wave * NC * 16 + col) * 2 + 1] = l;
    }
    float* dst = o_sh + (wave * NC * 16 + col) * LDO + 4 * q4;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      *reinterpret_cast<f32x4*>(dst + 16 * mt) = acc[c][mt];
    }
  }
  __syncthreads();
  // One wavefront finishes one packed row, VEC dims a lane.
  for (int col = wave; col < cols_live; col += 4) {
    float mw[4], lw[4], ow[4][VEC], o[VEC], L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      mw[w] = ml_sh[(w * NC * 16 + col) * 2];
      lw[w] = ml_sh[(w * NC * 16 + col) * 2 + 1];
#pragma unroll
      for (int e = 0; e < VEC; ++e) ow[w][e] = o_sh[(w * NC * 16 + col) * LDO + VEC * lane + e];
    }
    const float M = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = shaped_share(mw[w], M);
      L += f * lw[w];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] += ow[w][e] * f;
    }
    if (tile.part >= 0) {
      const size_t rec = (size_t(tile.part) * a.Hkv + kvh) * a.cols + col;
#pragma unroll
      for (int e = 0; e < VEC; ++e) a.parts_o[rec * HD + VEC * lane + e] = o[e];
      if (lane == 0) {
        a.parts_ml[rec * 2] = M;
        a.parts_ml[rec * 2 + 1] = L;
      }
    } else {
      const int m = col / a.G, hg = col - m * a.G;
      const float f = shaped_inverse(L);
      uint16_t* const to = a.O + size_t(tile.r0 + m) * a.q_ld + size_t(kvh * a.G + hg) * HD + VEC * lane;
#pragma unroll
      for (int e = 0; e < VEC; e += 2) *reinterpret_cast<uint32_t*>(to + e) = pack2<DT>(o[e] * f, o[e + 1] * f);
    }
  }
}

// Merge of the partial records of a split tile and the one rounding. Bound by the records' bytes, and for few rows by the latency of their
// loads. W wavefronts share one (job, row, head), taking its records round robin and meeting in LDS: 4 where groups have many
// records, else one, which keeps the records of four outputs in flight per workgroup.
template <int DT, int HD, int W>
__global__ __launch_bounds__(256) void attn_shaped_merge_kernel(const ShapedArgs a, const esp_combine* jobs) {
  constexpr int VEC = HD / 64;
  __shared__ float o_sh[W > 1 ? W : 1][W > 1 ? HD : 1];
  __shared__ float ml_sh[W > 1 ? W : 1][2];
  const esp_combine job = jobs[blockIdx.y];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int out = W > 1 ? int(blockIdx.x) : int(blockIdx.x) * 4 + wave;
  const int r = out / a.H, h = out - r * a.H;
  if (r >= job.rows) return;  // (for W > 1 the whole workgroup)
  const int kvh = h / a.G, col = r * a.G + h - kvh * a.G;
  const size_t step = size_t(a.Hkv) * a.cols;  // records from one part to the next
  float M = -INFINITY, L = 0.0f, o[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) o[e] = 0.0f;
  const size_t rec0 = (size_t(job.part0) * a.Hkv + kvh) * a.cols + col;
  for (int s = W > 1 ? wave : 0; s < job.nparts; s += 4 * W) {
    float mN[4], lN[4], oN[4][VEC];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // all loads before the first use; slots past the last record weigh nothing
      const size_t rec = rec0 + size_t(s + W * i < job.nparts ? s + W * i : s) * step;
      mN[i] = a.parts_ml[rec * 2];
      lN[i] = a.parts_ml[rec * 2 + 1];
#pragma unroll
      for (int e = 0; e < VEC; ++e) oN[i][e] = a.parts_o[rec * HD + VEC * lane + e];
    }
#pragma unroll
    for (int i = 1; i < 4; ++i) {  // (zeros, not a weight of zero: what is read again there may be infinite)
      const bool in = s + W * i < job.nparts;
      mN[i] = in ? mN[i] : -INFINITY;
      lN[i] = in ? lN[i] : 0.0f;
#pragma unroll
      for (int e = 0; e < VEC; ++e) oN[i][e] = in ? oN[i][e] : 0.0f;
    }
    float Mn = M;
#pragma unroll
    for (int i = 0; i < 4; ++i) Mn = fmaxf(Mn, mN[i]);
    const float c = shaped_share(M, Mn);
    L *= c;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] *= c;
    M = Mn;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = shaped_share(mN[i], Mn);
      L += w * lN[i];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] += oN[i][e] * w;
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) o_sh[wave][VEC * lane + e] = o[e];
    if (lane == 0) {
      ml_sh[wave][0] = M;
      ml_sh[wave][1] = L;
    }
    __syncthreads();
    if (wave != 0) return;
    M = ml_sh[0][0];
#pragma unroll
    for (int w = 1; w < W; ++w) M = fmaxf(M, ml_sh[w][0]);
    L = 0.0f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = shaped_share(ml_sh[w][0], M);
      L += f * ml_sh[w][1];
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[e] += o_sh[w][VEC * lane + e] * f;
    }
  }
  const float f = shaped_inverse(L);
  uint16_t* const to = a.O + size_t(job.r0 + r) * a.q_ld + size_t(h) * HD + VEC * lane;
#pragma unroll
  for (int e = 0; e < VEC; e += 2) *reinterpret_cast<uint32_t*>(to + e) = pack2<DT>(o[e] * f, o[e + 1] * f);
}

namespace {

constexpr size_t stream_smem(int HD, int NC) { return size_t(4 * NC * 16) * (HD + 4 + 2) * sizeof(float); }

template <int DT, int HD, int NC>
hipError_t allow_stream() {
  const hipError_t e = allow_dynamic_lds<attn_shaped_stream_kernel<DT, HD, NC, false>>(stream_smem(HD, NC));
  return e == hipSuccess ? allow_dynamic_lds<attn_shaped_stream_kernel<DT, HD, NC, true>>(stream_smem(HD, NC)) : e;
}

template <int DT>
hipError_t allow_streams() {
  hipError_t e = allow_stream<DT, 128, 1>();
  if (e == hipSuccess) e = allow_stream<DT, 128, 2>();
  if (e == hipSuccess) e = allow_stream<DT, 256, 1>();
  return e;
}

template <int DT, int HD, int NC, bool CAP>
hipError_t launch_stream_c(const ShapedArgs& a, int n_tiles, hipStream_t st) {
  constexpr size_t smem = stream_smem(HD, NC);
  constexpr auto k = attn_shaped_stream_kernel<DT, HD, NC, CAP>;
  const hipError_t e = allow_dynamic_lds<k>(smem);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(unsigned(a.Hkv), unsigned(n_tiles)), dim3(256), smem, st, a);
  return hipGetLastError();
}

template <int DT, int HD, int NC>
hipError_t launch_stream_t(const ShapedArgs& a, int n_tiles, hipStream_t st) {
  return a.cap_log2 > 0.0f ? launch_stream_c<DT, HD, NC, true>(a, n_tiles, st) : launch_stream_c<DT, HD, NC, false>(a, n_tiles, st);
}

// Pass and merge with one wavefront an output and with four, us: 16 parts of one tile 9.8 and 8.3, 63 of one 24.4 and 18.5 (of 24 rows 37 and 31), 64 of
// eight 27.0 and 26.6, 54 of eighteen 89.7 and 90.1. (2048 workgroups of four wavefronts are what the chip holds.)
template <int DT, int HD>
void launch_merge_t(const ShapedArgs& a, const esp_combine* jobs, int n_jobs, int n_parts, hipStream_t st) {
  const unsigned outs = unsigned(a.R * a.H), jobs_n = unsigned(n_jobs);
  if (n_parts > 4 * n_jobs && size_t(outs) * n_jobs < 2048)
    hipLaunchKernelGGL((attn_shaped_merge_kernel<DT, HD, 4>), dim3(outs, jobs_n), dim3(256), 0, st, a, jobs);
  else
    hipLaunchKernelGGL((attn_shaped_merge_kernel<DT, HD, 1>), dim3((outs + 3) / 4, jobs_n), dim3(256), 0, st, a, jobs);
}

}  // namespace

hipError_t shaped_init_attributes() {
  const hipError_t e = allow_streams<ESP_F16>();
  return e == hipSuccess ? allow_streams<ESP_BF16>() : e;
}

// a.cols <= 16 shaped_family and n_tiles <= 65535: the caller has checked.
hipError_t launch_shaped_stream(int dt, int HD, const ShapedArgs& a, int n_tiles, hipStream_t st) {
  if (HD == 256) return dt == ESP_F16 ? launch_stream_t<ESP_F16, 256, 1>(a, n_tiles, st) : launch_stream_t<ESP_BF16, 256, 1>(a, n_tiles, st);
  if (a.cols <= 16) return dt == ESP_F16 ? launch_stream_t<ESP_F16, 128, 1>(a, n_tiles, st) : launch_stream_t<ESP_BF16, 128, 1>(a, n_tiles, st);
  return dt == ESP_F16 ? launch_stream_t<ESP_F16, 128, 2>(a, n_tiles, st) : launch_stream_t<ESP_BF16, 128, 2>(a, n_tiles, st);
}

// n_jobs <= 65535: the caller has checked.
hipError_t launch_shaped_merge(int dt, int HD, const ShapedArgs& a, const esp_combine* jobs, int n_jobs, int n_parts, hipStream_t st) {
  if (HD == 256) dt == ESP_F16 ? launch_merge_t<ESP_F16, 256>(a, jobs, n_jobs, n_parts, st) : launch_merge_t<ESP_BF16, 256>(a, jobs, n_jobs, n_parts, st);
  else dt == ESP_F16 ? launch_merge_t<ESP_F16, 128>(a, jobs, n_jobs, n_parts, st) : launch_merge_t<ESP_BF16, 128>(a, jobs, n_jobs, n_parts, st);
  return hipGetLastError();
}

}  // namespace esp
