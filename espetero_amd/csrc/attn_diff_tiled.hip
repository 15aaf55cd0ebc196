// Differential attention (attn_diff.hip says what it computes) for passes with many rows: prompts, chunks, wide drafts.
//
// Bound by the matrix cores: 1536 operations for every pair of query heads, row and visible key. One workgroup is one tile and one KV
// pair; the tile's rows times the G query pairs of the KV pair are up to 128 packed rows (row in tile * G + query pair), so that
// K and V are staged once for all of them and a causal tile's rows lie close together. 8 wavefronts: wavefront w works on map w % 2
// of the 32 packed rows w / 2. Per 32 keys it computes
//   S^T[32 keys][32 rows] = K_map . Q_map^T      A = K from LDS, B = Q^T in registers
//   P^T = exp2(S^T - m)                          registers; the D layout of S^T is the B layout of P^T
//   O^T[256][32 rows]    += V^T . P^T            A = V^T from LDS, both maps read the same values
// with v_mfma_f32_32x32x16 and P . V one stage behind S. After the last key the second map's wavefronts hand their output over
// through LDS, and the first map's take the difference, the norm and the one rounding.
//
// LDS: a ring of 4 stages of 32 keys, 32 KB each: K of both heads, V^T of both heads, loaded straight from the pool
// (global_load_lds) three stages ahead. K: the 16-byte chunk c of row r lies at c ^ (pi(r) & 15), pi swapping bits 2 and 3;
// V^T: per sub-block of 16 keys and group of 32 dims [half of the keys][32 dims][8 keys], the order in which the lanes of a P . V
// operand read it. Neither side has bank conflicts.
#include "diff_math.hpp"
#include "lds_direct.hpp"

namespace esp {

namespace {
constexpr int kRing = 4, kStage = 32 * 1024;  // stages; bytes of one
constexpr size_t kDiffTiledLds = size_t(kRing) * kStage + 64;  // and 16 ints behind the ring
constexpr float kSlack = 8.0f;  // a row's reference moves when a score exceeds it by more (log2 units): P stays below 2^8
}  // namespace

template <int DT>
__global__ __launch_bounds__(512, 2) void attn_diff_tiled_kernel(const DiffArgs a) {
  constexpr int HD = kDiffHD, VD = kDiffVD, NT = VD / 32, KS = HD / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const uint32_t lds_base = uint32_t(uintptr_t(lds));
  const int j = blockIdx.x;  // KV pair
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hb = lane >> 5, map = wave & 1, col0 = 32 * (wave >> 1);
  const esp_tile tile = a.tiles[gridDim.y - 1 - blockIdx.y];  // last to first: a causal pass's longest tiles start first
  const esp_tree tree = a.trees[tile.tree];
  const int table = tile.pad > 0 ? tile.pad - 1 : tree.table;
  const DiffRange rg = diff_range(tile, tree, a.R, a.window);
  const int cols_live = rg.rows * a.G;

  // ---- this lane's packed row
  const int col = col0 + l32;
  const bool ok = col < cols_live;
  const int m = ok ? col / a.G : 0, hg = ok ? col - m * a.G : 0;
  const int qpos = tree.P + rg.rr0 + m;
  u32x4 qf[KS];
  {
    const uint16_t* qp = a.Q + size_t(tile.r0 + m) * a.q_ld + size_t(2 * (j * a.G + hg) + map) * HD + 8 * hb;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(qp + 16 * ks);
  }

  // ---- stages of 32 keys from the sub-block of the first key on; which of them this wavefront's rows see, and which whole
  const int s0 = rg.lo & ~15;
  const int n_st = rg.hi > rg.lo ? (rg.hi - s0 + 31) >> 5 : 0;
  int v0 = 0, v1 = 0, f0 = 0, f1 = 0;  // stages [v0, v1) hold keys that some row sees, [f0, f1) only keys that all see
  int w0 = 0, w1 = 0;                  // [w0, w1) only keys that all rows of the tile see
  if (n_st && col0 < cols_live) {
    const int q_first = tree.P + rg.rr0 + col0 / a.G, q_last = tree.P + rg.rr0 + (min(col0 + 32, cols_live) - 1) / a.G;
    const int some_lo = a.window > 0 ? max(rg.lo, q_first - a.window + 1) : rg.lo, some_hi = min(rg.hi, q_last + 1);
    const int all_lo = a.window > 0 ? max(rg.lo, q_last - a.window + 1) : rg.lo, all_hi = min(rg.hi, q_first + 1);
    v0 = (some_lo - s0) >> 5;
    v1 = max(v0, (some_hi - s0 + 31) >> 5);
    f0 = (all_lo - s0 + 31) >> 5;
    f1 = max(f0, (all_hi - s0) >> 5);
  }
  if (n_st) {
    const int q_last = tree.P + rg.rr0 + rg.rows - 1;
    w0 = ((a.window > 0 ? max(rg.lo, q_last - a.window + 1) : rg.lo) - s0 + 31) >> 5;
    w1 = max(w0, (min(rg.hi, tree.P + rg.rr0 + 1) - s0) >> 5);
  }

  // ---- staging: wavefront w loads sub-block w % 2 of K1, K2, V1 or V2 (w / 2) of every stage
  const int kind = wave >> 1, last_sub = rg.hi > rg.lo ? (rg.hi - 1) & ~15 : s0;
  const size_t head = size_t(2 * a.bt * HD);
  uint32_t voff[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * i + (lane >> 4);
    voff[i] = kind < 2 ? uint32_t((lane >> 4) * 256 + (((lane & 15) ^ swap23(r)) << 4)) : uint32_t((2 * l32 + hb) << 4);
  }
  const uint32_t dst = lds_base + wave * 4096;
  auto stage = [&](int h) {
    const int key = min(s0 + 32 * h + 16 * (wave & 1), last_sub);  // past the range: its last sub-block again
    const int t0 = key % a.bt;
    const uint16_t* hb_ = a.pool + diff_head_base(a, diff_block(a, table, key), 2 * j) + (kind & 1) * head;
    const uint16_t* src = kind < 2 ? hb_ + t0 * HD : hb_ + vt_elem(a.bt, HD, t0, 0);
    load_to_lds16_x4(src, voff[0], voff[1], voff[2], voff[3], dst + uint32_t(h % kRing) * kStage);
  };
  // Runs in a stage: K of head 0 sub-block 0, 1, K of head 1, V^T of head 0, V^T of head 1; 4 KB each.
  using lds_u32x4 = const __attribute__((address_space(3))) u32x4;
  auto lds_read = [&](uint32_t at) { return *reinterpret_cast<lds_u32x4*>(at); };
  const int prow = swap23(l32);  // the lane with S^T row l32 reads this key of the stage
  const uint32_t k_at = lds_base + map * 8192 + prow * 256;
  const uint32_t v_at = lds_base + 16384 + lane * 16;

  f32x16 acc[NT];
  float m_ref = -INFINITY, l_run = 0.0f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt] = f32x16{};
  u32x4 P[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};

  auto scores = [&](int h) {
    const uint32_t at = k_at + uint32_t(h % kRing) * kStage;
    f32x16 s{};
    u32x4 k[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k[ks] = lds_read(at + (((2 * ks + hb) ^ (l32 & 15)) << 4));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma32x16<DT>(k[ks], qf[ks], s);
    return s;
  };
  auto pv = [&](int h) {
    const uint32_t at = v_at + uint32_t(h % kRing) * kStage;
    u32x4 v[2][4];
    auto fetch = [&](int g) {  // of 4 groups: sub-block g / 2, dims 128 (g % 2) ..
#pragma unroll
      for (int i = 0; i < 4; ++i) v[g & 1][i] = lds_read(at + (g & 1) * 8192 + (g >> 1) * 4096 + i * 1024);
    };
    fetch(0);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (g < 3) fetch(g + 1);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[4 * (g & 1) + i] = mfma32x16<DT>(v[g & 1][i], P[g >> 1], acc[4 * (g & 1) + i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Lane l holds of S^T, at index 8 sb + i, key 16 sb + 8 hb + i of the stage.
  auto key_of = [&](int h, int sb, int i) { return s0 + 32 * h + 16 * sb + 8 * hb + i; };
  auto in_range = [&](int k0) {  // the bits of two keys' values
    return (k0 >= rg.lo && k0 < rg.hi ? 0xffffu : 0u) | (k0 + 1 >= rg.lo && k0 + 1 < rg.hi ? 0xffff0000u : 0u);
  };
  // Values of a stage with keys that some row does not see, by the wavefront that has staged them: those outside the range may be
  // memory never written, and infinite values of keys that only other rows see must not meet a zero weight. Both become zeros; where
  // there were any of the latter, `bad` says so and marks() adds them to the rows that see them.
  int* const bad = reinterpret_cast<int*>(lds + kRing * kStage);  // [stage of the ring][staging wavefront of the four]
  auto mend = [&](int h) {
    uint32_t found = 0;
    char* const mine = lds + (h % kRing) * kStage + wave * 4096 + lane * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 v = *reinterpret_cast<const u32x4*>(mine + i * 1024);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] &= in_range(key_of(h, wave & 1, 2 * e));
        const uint32_t nf = not_finite2<DT>(v[e]);
        found |= nf;
        v[e] &= ~nf;
      }
      *reinterpret_cast<u32x4*>(mine + i * 1024) = v;
    }
    const bool any = __any(found != 0);
    if (lane == 0) bad[4 * (h % kRing) + (wave & 3)] = any;
  };
  auto marks = [&](int h) {
    const uint16_t* src[2];
#pragma unroll
    for (int sb = 0; sb < 2; ++sb) {
      const int key = min(s0 + 32 * h + 16 * sb, last_sub);
      src[sb] = a.pool + diff_head_base(a, diff_block(a, table, key), 2 * j) + vt_elem(a.bt, HD, key % a.bt, l32) + 8 * hb;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int neg = 0; neg < 2; ++neg) {
        f32x16 seen{};
#pragma unroll
        for (int sb = 0; sb < 2; ++sb) {
          u32x4 v = *reinterpret_cast<const u32x4*>(src[sb] + (nt >> 2) * head + 32 * (nt & 3) * kVtDim);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = not_finite_marks<DT>(v[e] & in_range(key_of(h, sb, 2 * e)), neg != 0);
          seen = mfma32x16<DT>(v, P[sb], seen);
        }
        mfma_settle(seen);
        mfma_settle(acc[nt]);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (seen[e] > 0.0f) acc[nt][e] += neg ? -INFINITY : INFINITY;
        __builtin_amdgcn_sched_barrier(0);
      }
  };

  if (n_st > 0) stage(0);
  if (n_st > 1) stage(1);
  if (n_st > 2) stage(2);
  // One turn more than stages: turn h has S of stage h and P . V of stage h - 1.
  for (int h = 0; h <= n_st; ++h) {
    // Stage h is in LDS for everybody, and everybody is done with stage h - 2, whose place stage h + 2 takes.
    const int behind = min(n_st, h + 2) - (h + 1);  // stages requested behind stage h, 4 loads each
    if (behind >= 1) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (wave >= 4 && h < n_st && (h < w0 || h >= w1)) {
      mend(h);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (h >= 1 && h + 2 < n_st) stage(h + 2);
    const bool do_s = h >= v0 && h < v1, do_pv = h - 1 >= v0 && h - 1 < v1;
    const bool s_full = h >= f0 && h < f1, pv_full = h - 1 >= w0 && h - 1 < w1;
    f32x16 s{};
    float c = 1.0f;
    bool move = false;
    if (do_s) {
      s = scores(h);
      mfma_settle(s);
      if (!s_full) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = key_of(h, e >> 3, e & 7);
          bool vis = key >= rg.lo && key < rg.hi && key <= qpos;
          if (a.window > 0) vis = vis && qpos - key < a.window;
          s[e] = vis ? s[e] : -INFINITY;
        }
      }
      float mx = s[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
      mx = fmaxf(mx, __shfl_xor(mx, 32)) * a.scale_log2;
      const bool up = mx > m_ref + kSlack;  // from -inf on: the first key that the row sees
      c = up ? fast_exp2(m_ref - mx) : 1.0f;
      m_ref = up ? mx : m_ref;
      move = __any(up);
    }
    if (do_pv) {
      pv(h - 1);
      if (!pv_full) {
        const int* b = bad + 4 * ((h - 1) % kRing);
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(b[0] | b[1] | b[2] | b[3]), 0)) marks(h - 1);
      }
    }
    if (do_s) {
      if (__builtin_expect(move, 0)) {
        l_run *= c;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mfma_settle(acc[nt]);
          acc[nt] *= c;
        }
      }
      const float off = m_ref == -INFINITY ? 0.0f : m_ref;
      float p[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        p[e] = fast_exp2(s[e] * a.scale_log2 - off);
        l_run += p[e];
      }
#pragma unroll
      for (int sb = 0; sb < 2; ++sb)
        P[sb] = u32x4{pack2<DT>(p[8 * sb], p[8 * sb + 1]), pack2<DT>(p[8 * sb + 2], p[8 * sb + 3]), pack2<DT>(p[8 * sb + 4], p[8 * sb + 5]),
                      pack2<DT>(p[8 * sb + 6], p[8 * sb + 7])};
    }
  }

  // ---- the row's end
  float l = l_run + __shfl_xor(l_run, 32);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) mfma_settle(acc[nt]);
  if (tile.part >= 0) {  // a partial record: dims 32 nt + 8 i + 4 hb .. + 3 of this lane's packed row
    if (!ok) return;
    const size_t rec = ((size_t(tile.part) * (a.Hkv / 2) + j) * 2 + map) * a.cols + col;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(a.parts_o + rec * VD + 32 * nt + 8 * i + 4 * hb) = f32x4{acc[nt][4 * i], acc[nt][4 * i + 1], acc[nt][4 * i + 2], acc[nt][4 * i + 3]};
    if (hb == 0) {
      a.parts_ml[rec * 2] = m_ref;
      a.parts_ml[rec * 2 + 1] = l;
    }
    return;
  }
  __syncthreads();  // the ring is free
  f32x4* const sh = reinterpret_cast<f32x4*>(lds + (wave >> 1) * 32768) + lane;  // [32 groups of 4 dims][64 lanes]
  const int pair = j * a.G + hg;
  if (map == 1) {
    const float i2 = (l > 0.0f ? 1.0f / l : 0.0f) * a.weight[pair];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sh[64 * (4 * nt + i)] = f32x4{acc[nt][4 * i] * i2, acc[nt][4 * i + 1] * i2, acc[nt][4 * i + 2] * i2, acc[nt][4 * i + 3] * i2};
  }
  __syncthreads();
  if (map == 1) return;
  const float i1 = l > 0.0f ? 1.0f / l : 0.0f;
  float ss = 0.0f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4 o2 = sh[64 * (4 * nt + i)];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float o = acc[nt][4 * i + e] * i1 - o2[e];
        acc[nt][4 * i + e] = o;
        ss += o * o;
      }
    }
  ss += __shfl_xor(ss, 32);
  if (!ok) return;
  const float f = a.norm_w ? a.factor * rsqrtf(ss * (1.0f / VD) + a.eps) : a.factor;
  uint16_t* const to = a.O + size_t(tile.r0 + m) * a.q_ld + size_t(pair) * VD;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = 32 * nt + 8 * i + 4 * hb;
      f32x4 w = {f, f, f, f};
      if (a.norm_w) w *= *reinterpret_cast<const f32x4*>(a.norm_w + d);
      *reinterpret_cast<u32x2*>(to + d) = u32x2{pack2<DT>(acc[nt][4 * i] * w[0], acc[nt][4 * i + 1] * w[1]),
                                                pack2<DT>(acc[nt][4 * i + 2] * w[2], acc[nt][4 * i + 3] * w[3])};
    }
}

hipError_t diff_tiled_init_attributes() {
  const hipError_t e = allow_dynamic_lds<attn_diff_tiled_kernel<ESP_F16>>(kDiffTiledLds);
  return e == hipSuccess ? allow_dynamic_lds<attn_diff_tiled_kernel<ESP_BF16>>(kDiffTiledLds) : e;
}

template <int DT>
static hipError_t launch_diff_tiled_t(const DiffArgs& a, int n_tiles, hipStream_t st) {
  constexpr auto k = attn_diff_tiled_kernel<DT>;
  const hipError_t e = allow_dynamic_lds<k>(kDiffTiledLds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(unsigned(a.Hkv / 2), unsigned(n_tiles)), dim3(512), kDiffTiledLds, st, a);
  return hipGetLastError();
}

// a.cols <= 128 and n_tiles <= 65535: the caller has checked.
hipError_t launch_diff_tiled(int dt, const DiffArgs& a, int n_tiles, hipStream_t st) {
  return dt == ESP_F16 ? launch_diff_tiled_t<ESP_F16>(a, n_tiles, st) : launch_diff_tiled_t<ESP_BF16>(a, n_tiles, st);
}

}  // namespace esp
