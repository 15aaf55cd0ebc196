// Differential attention over the paged pool. A pair of query heads (2 i, 2 i + 1) reads a pair of KV heads (2 j, 2 j + 1):
// head 2 i scores the keys of KV head 2 j, head 2 i + 1 those of 2 j + 1, both maps weigh the same 256-dim values, the two KV
// heads' values side by side, and
//   O = factor * norm( softmax(scale q1 K1^T) V - weight[i] * softmax(scale q2 K2^T) V ).
// The rows of the pass are in the pool (appended before the call); row r of a tree sees the keys 0 .. P + r, the last `window` of
// them on a sliding layer.
//
// Streaming kernel: decode and short trees. Bound by HBM: every visible key's 1 KB per KV pair (K1, K2 and V, 16 bits) is read
// once for both maps and all G query pairs. One workgroup is one tile and one KV pair; up to 8 packed rows (row in tile * G + query
// pair) of both maps share the 16 columns of a matrix tile: columns 0 .. 7 are the first map's, 8 .. 15 the second's. Of the products
// with K1 and with K2 a lane keeps its own map's, one softmax serves both, and so does one product P . V. A wavefront takes 16-key
// units round robin straight from HBM (64 registers of operands: 16 KB per wavefront and set) with the next unit's loads in flight.
// 24 users of 300 to 9000 keys, 32 / 8 heads: 96 us, 5.6 TB/s; four documents of 50000 to 60000, 32 / 4 heads: 79 us, 5.9 TB/s (a copy
// reaches 4.9, a bare read 6.8), and what is read from memory is the visible keys' bytes to 0.5 %; one user of 1000 keys: 9.7 us, its
// cuts' hops and the merge's launch.
#include "diff_math.hpp"

namespace esp {

namespace {

struct DiffUnit {  // 16 keys: K of both heads, V^T of both heads
  u32x4 k[2][4];   // [map][32-dim group]: key = lane % 16, dims 32 kk + 8 (lane / 16) ..
  u32x2 v[16];     // [16-dim group of the 256]: dim = 16 mt + lane % 16, keys 4 (lane / 16) ..
};

}  // namespace

// NC: column tiles of 8 packed rows (x 2 maps).
template <int DT, int NC>
__global__ __launch_bounds__(256, 1) void attn_diff_stream_kernel(const DiffArgs a) {
  constexpr int HD = kDiffHD, VD = kDiffVD, MT = VD / 16, LDO = VD + 4;
  extern __shared__ float smem[];  // [4 wavefronts][NC * 16 columns][LDO] O, then [4][NC * 16][2] m, l
  const int j = blockIdx.x;        // KV pair
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c16 = lane & 15, q4 = lane >> 4, map = c16 >> 3;
  const esp_tile tile = a.tiles[blockIdx.y];
  const esp_tree tree = a.trees[tile.tree];
  const int table = tile.pad > 0 ? tile.pad - 1 : tree.table;
  const DiffRange rg = diff_range(tile, tree, a.R, a.window);
  const int cols_live = rg.rows * a.G;

  // ---- this lane's packed rows: Q operands and positions
  u32x4 qf[NC][4];
  int qpos[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = 8 * c + (c16 & 7);
    const bool ok = col < cols_live;
    const int m = ok ? col / a.G : 0, hg = ok ? col - m * a.G : 0;
    qpos[c] = tree.P + rg.rr0 + m;
    const uint16_t* qp = a.Q + size_t(tile.r0 + m) * a.q_ld + size_t(2 * (j * a.G + hg) + map) * HD + 8 * q4;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) qf[c][kk] = ok ? *reinterpret_cast<const u32x4*>(qp + 32 * kk) : u32x4{0, 0, 0, 0};
  }

  // ---- 16-key units; interior ones are seen whole by every row of the tile
  const int u_lo = rg.lo >> 4, u_hi = (rg.hi + 15) >> 4;  // all units [u_lo, u_hi), none if the range is empty
  const int n_units = rg.hi > rg.lo ? u_hi - u_lo : 0;
  int full_lo = rg.lo;
  const int q_first = tree.P + rg.rr0, q_last = q_first + rg.rows - 1;
  if (a.window > 0) full_lo = max(full_lo, q_last - a.window + 1);
  const int full_hi = min(rg.hi, q_first + 1);
  int ui0 = u_lo, ui1 = u_lo;
  if (n_units) {
    ui0 = min((full_lo + 15) >> 4, u_hi);
    ui1 = max(ui0, full_hi >> 4);
  }

  f32x4 acc[NC][MT];
  float m_run[NC], l_run[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m_run[c] = -INFINITY;
    l_run[c] = 0.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[c][mt] = f32x4{0, 0, 0, 0};
  }

  // Where a unit's operands lie: one address for the block's KV pair, everything else are offsets from it.
  const uint32_t lane_k = uint32_t(c16 * HD + 8 * q4) * 2, lane_v = uint32_t(c16 * kVtDim + 4 * q4) * 2;
  const uint32_t head = uint32_t(2 * a.bt * HD) * 2, to_v = uint32_t(a.bt * HD) * 2;  // bytes of one (block, KV head); from its K to its V^T
  const uint64_t block_bytes = uint64_t(a.Hkv) * head;
  const char* const pool = reinterpret_cast<const char*>(a.pool + a.kv_base) + uint64_t(2 * j) * head;
  auto block_of = [&](int u) {  // (a sub-block of V^T starts as far behind the first as its first token's K row does)
    const int key = u << 4, bi = key / a.bt;
    return pool + uint64_t(uint32_t(diff_block(a, table, bi))) * block_bytes + uint32_t(key - bi * a.bt) * (HD * 2);
  };
  auto load = [&](int u, DiffUnit& U) {
    const char* const base = block_of(u);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* const kp = base + h * head;
      const char* const vp = kp + to_v;
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) U.k[h][kk] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kp + lane_k + 64 * kk));
#pragma unroll
      for (int mt = 0; mt < 8; ++mt) U.v[8 * h + mt] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vp + lane_v + 32 * kVtDim * mt));
    }
  };
  auto scores = [&](const DiffUnit& U, f32x4 (&s)[NC]) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      f32x4 of[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
#pragma unroll
        for (int h = 0; h < 2; ++h) of[h] = mfma16x32<DT>(U.k[h][kk], qf[c][kk], of[h]);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[c][e] = map ? of[1][e] : of[0][e];
    }
  };
  // Online softmax over scores x (log2 units, -inf where masked), then O^T += V^T . P^T. The matrix product takes P in the storage
  // type: as the sum of two such numbers, 16 bits or more, since one alone makes the output 1.4 times as inexact as its own rounding
  // does and the second product waits for memory anyway. p: the weights before that.
  auto softmax_pv = [&](const DiffUnit& U, const f32x4 (&x)[NC], f32x4 (&p)[NC]) {
    bool any_change = false;
    float corr[NC];
    u32x2 pb[NC], pl[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float mx = fmaxf(fmaxf(x[c][0], x[c][1]), fmaxf(x[c][2], x[c][3]));
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m_run[c], mx);
      const float m_safe = (m_new == -INFINITY) ? 0.0f : m_new;
      corr[c] = fast_exp2(m_run[c] - m_safe);
      any_change = any_change || (m_new > m_run[c]);
      m_run[c] = m_new;
#pragma unroll
      for (int e = 0; e < 4; ++e) p[c][e] = fast_exp2(x[c][e] - m_safe);
      l_run[c] = l_run[c] * corr[c] + (p[c][0] + p[c][1] + p[c][2] + p[c][3]);
      pb[c] = u32x2{pack2<DT>(p[c][0], p[c][1]), pack2<DT>(p[c][2], p[c][3])};
      pl[c] = u32x2{pack2<DT>(p[c][0] - unpack_lo<DT>(pb[c].x), p[c][1] - unpack_hi<DT>(pb[c].x)),
                    pack2<DT>(p[c][2] - unpack_lo<DT>(pb[c].y), p[c][3] - unpack_hi<DT>(pb[c].y))};
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
  auto interior = [&](const DiffUnit& U) {
    f32x4 s[NC], p[NC];
    scores(U, s);
#pragma unroll
    for (int c = 0; c < NC; ++c) s[c] *= a.scale_log2;
    softmax_pv(U, s, p);
  };
  // A unit with keys that some row does not see.
  auto edge = [&](int u, DiffUnit& U) {
    // Keys outside the range may be memory never written: their V must not reach the products (0 * NaN).
    const int jv = (u << 4) + 4 * q4;
    uint32_t in[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) in[e] = (jv + e >= rg.lo && jv + e < rg.hi) ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
    uint32_t bad = 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      U.v[mt].x &= in[0] | in[1];
      U.v[mt].y &= in[2] | in[3];
      bad |= not_finite2<DT>(U.v[mt].x) | not_finite2<DT>(U.v[mt].y);
    }
    // Nor may the infinite V of a key that one row sees reach a row that does not: such elements leave the product, and a product of
    // marks in their places says which rows see them.
    const bool rare = rg.rows > 1 && __any(bad != 0);
    if (rare) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        U.v[mt].x &= ~not_finite2<DT>(U.v[mt].x);
        U.v[mt].y &= ~not_finite2<DT>(U.v[mt].y);
      }
    }
    f32x4 s[NC], p[NC];
    scores(U, s);
#pragma unroll
    for (int c = 0; c < NC; ++c) mfma_settle(s[c]);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // The row sees the keys [from, from + n).
        const int from = a.window > 0 ? max(rg.lo, qpos[c] - a.window + 1) : rg.lo, n = max(0, min(rg.hi, qpos[c] + 1) - from);
        s[c][e] = uint32_t(jv + e - from) < uint32_t(n) ? s[c][e] * a.scale_log2 : -INFINITY;
      }
    softmax_pv(U, s, p);
    if (__builtin_expect(rare, 0)) {
      const char* const vp = block_of(u) + to_v + lane_v;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(vp + (mt >> 3) * head + 32 * kVtDim * (mt & 7));
        const uint32_t lo = v.x & (in[0] | in[1]), hi = v.y & (in[2] | in[3]);
#pragma unroll
        for (int neg = 0; neg < 2; ++neg)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const u32x2 pb = {pack2<DT>(p[c][0], p[c][1]), pack2<DT>(p[c][2], p[c][3])};
            f32x4 seen = mfma16x16<DT>(u32x2{not_finite_marks<DT>(lo, neg != 0), not_finite_marks<DT>(hi, neg != 0)}, pb, f32x4{0, 0, 0, 0});
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

  {
    DiffUnit U[2];
    const int n_int = ui1 - ui0, n_lo = ui0 - u_lo, n_edge = n_units - n_int;
    const int n_mine = n_int > wave ? (n_int - wave + 3) / 4 : 0;
    if (n_mine > 0) {
      const int u0 = ui0 + wave;
      load(u0, U[0]);
      int i = 0;
      for (; i + 2 < n_mine; i += 2) {
        load(u0 + 4 * (i + 1), U[1]);
        interior(U[0]);
        load(u0 + 4 * (i + 2), U[0]);
        interior(U[1]);
      }
      if (i + 2 == n_mine) {
        load(u0 + 4 * (i + 1), U[1]);
        interior(U[0]);
        interior(U[1]);
      } else {
        interior(U[0]);
      }
    }
    for (int i = (wave + 4 - n_int % 4) % 4; i < n_edge; i += 4) {  // go on with the round robin
      const int u = i < n_lo ? u_lo + i : ui1 + (i - n_lo);
      load(u, U[0]);
      edge(u, U[0]);
    }
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
      mfma_settle(acc[c][mt]);
      *reinterpret_cast<f32x4*>(dst + 16 * mt) = acc[c][mt];
    }
  }
  __syncthreads();
  // One wavefront finishes one packed row, 4 dims of both maps per lane.
  for (int col = wave; col < cols_live; col += 4) {
    f32x4 o[2];
    float M[2], L[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = (col >> 3) * 16 + 8 * h + (col & 7);
      float mw[4], lw[4];
      f32x4 ow[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        mw[w] = ml_sh[(w * NC * 16 + at) * 2];
        lw[w] = ml_sh[(w * NC * 16 + at) * 2 + 1];
        ow[w] = *reinterpret_cast<const f32x4*>(o_sh + (w * NC * 16 + at) * LDO + 4 * lane);
      }
      M[h] = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
      L[h] = 0.0f;
      o[h] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = mw[w] == -INFINITY ? 0.0f : fast_exp2(mw[w] - M[h]);
        L[h] += f * lw[w];
        o[h] += ow[w] * f;
      }
    }
    if (tile.part >= 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const size_t rec = ((size_t(tile.part) * (a.Hkv / 2) + j) * 2 + h) * a.cols + col;
        *reinterpret_cast<f32x4*>(a.parts_o + rec * VD + 4 * lane) = o[h];
        if (lane == 0) {
          a.parts_ml[rec * 2] = M[h];
          a.parts_ml[rec * 2 + 1] = L[h];
        }
      }
    } else {
      const int m = col / a.G, hg = col - m * a.G;
      diff_finish<DT>(a, tile.r0 + m, j * a.G + hg, lane, o[0], L[0], o[1], L[1]);
    }
  }
}

// Merge of the partial records of a split tile, then the difference, the norm and the one rounding. Bound by the records' bytes, 2 KB
// of fp32 each, and for few rows by the latency of their loads. W wavefronts share one (job, row, query pair), taking its records round
// robin and meeting in LDS: 4 where groups have many records, else one, which keeps the records of four outputs in flight per workgroup
// (126 parts of 128 packed rows, two a group: 27.1 us with four wavefronts an output, 15.6 with one).
template <int DT, int W>
__global__ __launch_bounds__(256) void attn_diff_merge_kernel(const DiffArgs a, const esp_combine* jobs) {
  constexpr int VD = kDiffVD;
  __shared__ __attribute__((aligned(16))) float o_sh[W > 1 ? W : 1][2][W > 1 ? VD : 4];
  __shared__ float ml_sh[W > 1 ? W : 1][2][2];
  const esp_combine job = jobs[blockIdx.y];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int pairs = a.H / 2, out = W > 1 ? int(blockIdx.x) : int(blockIdx.x) * 4 + wave;
  const int r = out / pairs, pair = out - r * pairs;
  if (r >= job.rows) return;  // (for W > 1 the whole workgroup)
  const int j = pair / a.G, col = r * a.G + pair - j * a.G;
  const size_t step = size_t(a.Hkv) * a.cols;  // records from one part to the next (Hkv / 2 pairs x 2 maps)
  float M[2] = {-INFINITY, -INFINITY}, L[2] = {0.0f, 0.0f};
  f32x4 o[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  const size_t rec0 = (size_t(job.part0) * (a.Hkv / 2) + j) * 2 * a.cols + col;
  for (int s = W > 1 ? wave : 0; s < job.nparts; s += 4 * W) {
    float mN[2][4], lN[2][4];
    f32x4 oN[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // all loads before the first use; slots past the last record weigh nothing
        const bool in = s + W * i < job.nparts;
        const size_t rec = rec0 + size_t(h) * a.cols + size_t(in ? s + W * i : s) * step;
        mN[h][i] = in ? a.parts_ml[rec * 2] : -INFINITY;
        lN[h][i] = a.parts_ml[rec * 2 + 1];
        oN[h][i] = *reinterpret_cast<const f32x4*>(a.parts_o + rec * VD + 4 * lane);
      }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float Mn = M[h];
#pragma unroll
      for (int i = 0; i < 4; ++i) Mn = fmaxf(Mn, mN[h][i]);
      const float c = M[h] == -INFINITY ? 0.0f : fast_exp2(M[h] - Mn);
      L[h] *= c;
      o[h] *= c;
      M[h] = Mn;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = mN[h][i] == -INFINITY ? 0.0f : fast_exp2(mN[h][i] - Mn);
        L[h] += w * lN[h][i];
        o[h] += oN[h][i] * w;
      }
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<f32x4*>(&o_sh[wave][h][4 * lane]) = o[h];
      if (lane == 0) {
        ml_sh[wave][h][0] = M[h];
        ml_sh[wave][h][1] = L[h];
      }
    }
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float Mn = ml_sh[0][h][0];
#pragma unroll
      for (int w = 1; w < W; ++w) Mn = fmaxf(Mn, ml_sh[w][h][0]);
      o[h] = f32x4{0, 0, 0, 0};
      L[h] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = ml_sh[w][h][0] == -INFINITY ? 0.0f : fast_exp2(ml_sh[w][h][0] - Mn);
        L[h] += f * ml_sh[w][h][1];
        o[h] += *reinterpret_cast<const f32x4*>(&o_sh[w][h][4 * lane]) * f;
      }
    }
  }
  diff_finish<DT>(a, job.r0 + r, pair, lane, o[0], L[0], o[1], L[1]);
}

static size_t diff_stream_smem(int NC) { return size_t(4 * NC * 16) * (kDiffVD + 4 + 2) * sizeof(float); }

hipError_t diff_init_attributes() {
  hipError_t e = allow_dynamic_lds<attn_diff_stream_kernel<ESP_F16, 1>>(diff_stream_smem(1));
  if (e == hipSuccess) e = allow_dynamic_lds<attn_diff_stream_kernel<ESP_F16, 2>>(diff_stream_smem(2));
  if (e == hipSuccess) e = allow_dynamic_lds<attn_diff_stream_kernel<ESP_BF16, 1>>(diff_stream_smem(1));
  if (e == hipSuccess) e = allow_dynamic_lds<attn_diff_stream_kernel<ESP_BF16, 2>>(diff_stream_smem(2));
  return e;
}

template <int DT, int NC>
static hipError_t launch_diff_stream_t(const DiffArgs& a, int n_tiles, hipStream_t st) {
  const size_t smem = diff_stream_smem(NC);
  constexpr auto k = attn_diff_stream_kernel<DT, NC>;
  const hipError_t e = allow_dynamic_lds<k>(smem);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(unsigned(a.Hkv / 2), unsigned(n_tiles)), dim3(256), smem, st, a);
  return hipGetLastError();
}

// a.cols <= 16 and n_tiles <= 65535: the caller has checked.
hipError_t launch_diff_stream(int dt, const DiffArgs& a, int n_tiles, hipStream_t st) {
  if (a.cols <= 8) return dt == ESP_F16 ? launch_diff_stream_t<ESP_F16, 1>(a, n_tiles, st) : launch_diff_stream_t<ESP_BF16, 1>(a, n_tiles, st);
  return dt == ESP_F16 ? launch_diff_stream_t<ESP_F16, 2>(a, n_tiles, st) : launch_diff_stream_t<ESP_BF16, 2>(a, n_tiles, st);
}

// n_jobs <= 65535: the caller has checked.
hipError_t launch_diff_merge(int dt, const DiffArgs& a, const esp_combine* jobs, int n_jobs, int n_parts, hipStream_t st) {
  const unsigned outs = unsigned(a.R * (a.H / 2)), jobs_n = unsigned(n_jobs);
  if (n_parts > 4 * n_jobs && size_t(outs) * n_jobs < 2048) {
    if (dt == ESP_F16) hipLaunchKernelGGL((attn_diff_merge_kernel<ESP_F16, 4>), dim3(outs, jobs_n), dim3(256), 0, st, a, jobs);
    else hipLaunchKernelGGL((attn_diff_merge_kernel<ESP_BF16, 4>), dim3(outs, jobs_n), dim3(256), 0, st, a, jobs);
  } else {
    if (dt == ESP_F16) hipLaunchKernelGGL((attn_diff_merge_kernel<ESP_F16, 1>), dim3((outs + 3) / 4, jobs_n), dim3(256), 0, st, a, jobs);
    else hipLaunchKernelGGL((attn_diff_merge_kernel<ESP_BF16, 1>), dim3((outs + 3) / 4, jobs_n), dim3(256), 0, st, a, jobs);
  }
  return hipGetLastError();
}

}  // namespace esp
