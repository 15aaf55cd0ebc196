// Attention with shaped scores (attn_shaped.hip says what it computes) for passes with many rows: prompts, chunks, wide drafts.
//
// Bound by the matrix cores and the vector units beside them: 4 head_dim operations for every query head, row and visible key, and one
// exponential for its weight, two more for a cap. One workgroup is one tile and one KV head; the tile's rows times the G
// query heads are up to 128 packed rows (row in tile * G + head of the group), 32 a wavefront. Per 32 keys a wavefront computes
//   S^T[32 keys][32 rows] = K . Q^T      A = K from LDS, B = Q^T in registers
//   P^T = exp2(shaped(S^T) - m)          registers; the D layout of S^T is the B layout of P^T
//   O^T[head_dim][32 rows] += V^T . P^T  A = V^T from LDS
// with v_mfma_f32_32x32x16 and P . V one stage behind S.
//
// LDS: a ring of 4 stages of 32 keys, K and V^T, loaded straight from the pool (global_load_lds) two stages ahead: wavefronts 0 and 1 load the
// two sub-blocks of K, 2 and 3 those of V^T. K: the 16-byte chunk c of row r lies at c ^ (pi(r) & 15), pi swapping bits 2 and 3; V^T: per
// sub-block of 16 keys and group of 32 dims [half of the keys][32 dims][8 keys], the order in which the lanes of a P . V operand read
// it. Neither side has bank conflicts. Nothing in the loop may load from memory but the stages (any such load's wait is a wait for them).
#include "lds_direct.hpp"
#include "rows_out.hpp"
#include "shaped_math.hpp"

namespace esp {

namespace {
constexpr int kRing = 4;
constexpr float kSlack = 8.0f;  // a row's reference moves when a score exceeds it by more (log2 units): P stays below 2^8

template <int HD>
struct TiledLds {
  static constexpr int kRun = 32 * HD;          // bytes of a sub-block of 16 keys of K or of V^T
  static constexpr int kStage = 4 * kRun;       // K 0, K 1, V^T 0, V^T 1
  static constexpr int kBad = kRing * kStage;   // 8 ints behind the ring; then a word per lane and 32 dims
  static constexpr int kMarks = kBad + 64;
  static constexpr int kBytes = kMarks + 4 * (HD / 32) * 256;
};

// The maximum over the two lanes that hold a row. (Of the builtin for this instruction the compiler keeps one result only; the two
// wait states are what it puts between a vector instruction and the exchange of its result.)
__device__ __forceinline__ float max_halves(float x) {
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}
}  // namespace

template <int DT, int HD, bool CAP>
__global__ __launch_bounds__(256, HD == 128 ? 2 : 1) void attn_shaped_tiled_kernel(const ShapedArgs a) {
  using L = TiledLds<HD>;
  constexpr int NT = HD / 32, KS = HD / 16, RB = HD * 2, LOADS = L::kRun / 1024;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const uint32_t lds_base = uint32_t(uintptr_t(lds));
  const int kvh = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hb = lane >> 5, col0 = 32 * wave;
  const esp_tile tile = a.tiles[gridDim.y - 1 - blockIdx.y];  // last to first: a causal pass's longest tiles start first
  const esp_tree tree = a.trees[tile.tree];
  const int table = tile.pad > 0 ? tile.pad - 1 : tree.table;
  const int rr0 = tile.r0 - tree.base, rows = min(a.R, tree.M - rr0), cols_live = rows * a.G;
  const int n_keys = tree.P + tree.M;

  // ---- this lane's packed row (of lanes behind the last one, that one's)
  struct Place {
    int m, hg;  // row in the tile, head of the group
  };
  auto place = [&](int l) {
    const int col = min(col0 + (l & 31), cols_live - 1), m = col / a.G;
    return Place{m, col - m * a.G};
  };
  u32x4 qf[KS];
  int qpos;
  Sight sight;
  float slope;
  {
    const Place pl = place(lane);
    qpos = tree.P + rr0 + pl.m;
    const uint16_t* qp = a.Q + size_t(tile.r0 + pl.m) * a.q_ld + size_t(kvh * a.G + pl.hg) * HD + 8 * hb;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4*>(qp + 16 * ks);
    sight = shaped_sight(a, tile.r0 + pl.m, qpos, n_keys);
    slope = a.slopes ? a.slopes[kvh * a.G + pl.hg] * kLog2e : 0.0f;
  }
  // What some and what all of a set of rows see: of this wavefront's and of the tile's.
  struct Seen {
    int some_from, some_end, all_from, all_end;
  };
  Seen mine{}, whole{};
  if (a.spans) {
    auto reduce = [](Seen s, int lanes) {
      for (int x = 1; x < lanes; x <<= 1) {
        s.some_from = min(s.some_from, __shfl_xor(s.some_from, x));
        s.some_end = max(s.some_end, __shfl_xor(s.some_end, x));
        s.all_from = max(s.all_from, __shfl_xor(s.all_from, x));
        s.all_end = min(s.all_end, __shfl_xor(s.all_end, x));
      }
      s.some_from = __builtin_amdgcn_readfirstlane(s.some_from), s.some_end = __builtin_amdgcn_readfirstlane(s.some_end);
      s.all_from = __builtin_amdgcn_readfirstlane(s.all_from), s.all_end = __builtin_amdgcn_readfirstlane(s.all_end);
      return s;
    };
    mine = reduce(Seen{sight.from, sight.end, sight.from, sight.end}, 32);
    const int m0 = min(lane, rows - 1), m1 = min(lane + 64, rows - 1);
    const Sight s0 = shaped_sight(a, tile.r0 + m0, tree.P + rr0 + m0, n_keys), s1 = shaped_sight(a, tile.r0 + m1, tree.P + rr0 + m1, n_keys);
    whole = reduce(Seen{min(s0.from, s1.from), max(s0.end, s1.end), max(s0.from, s1.from), min(s0.end, s1.end)}, 64);
  } else {
    auto of_rows = [&](int m0, int m1) {
      const int q0 = tree.P + rr0 + m0, q1 = tree.P + rr0 + m1;
      return Seen{a.window > 0 ? max(0, q0 - a.window + 1) : 0, q1 + 1, a.window > 0 ? max(0, q1 - a.window + 1) : 0, q0 + 1};
    };
    mine = of_rows(min(col0, cols_live - 1) / a.G, (min(col0 + 32, cols_live) - 1) / a.G);
    whole = of_rows(0, rows - 1);
  }
  const Sight rg = shaped_range(tile, tree, whole.some_from, whole.some_end);

  // ---- stages of 32 keys from the sub-block of the first key on; which of them this wavefront's rows see, and which whole
  const int s0 = rg.from & ~15;
  const int n_st = rg.end > rg.from ? (rg.end - s0 + 31) >> 5 : 0;
  int v0 = 0, v1 = 0, f0 = 0, f1 = 0;  // stages [v0, v1) hold keys that some row sees, [f0, f1) only keys that all see
  int w0 = 0, w1 = 0;                  // [w0, w1) only keys that all rows of the tile see
  if (n_st && col0 < cols_live) {
    const int some_lo = max(rg.from, mine.some_from), some_hi = min(rg.end, mine.some_end);
    const int all_lo = max(rg.from, mine.all_from), all_hi = min(rg.end, mine.all_end);
    if (some_hi > some_lo) {
      v0 = (some_lo - s0) >> 5;
      v1 = (some_hi - s0 + 31) >> 5;
      f0 = (all_lo - s0 + 31) >> 5;
      f1 = max(f0, (all_hi - s0) >> 5);
    }
  }
  if (n_st) {
    w0 = (max(rg.from, whole.all_from) - s0 + 31) >> 5;
    w1 = max(w0, (min(rg.end, whole.all_end) - s0) >> 5);
  }

  // ---- staging: wavefront w loads sub-block w % 2 of K or V (w / 2) of every stage
  const int kind = wave >> 1, last_sub = rg.end > rg.from ? (rg.end - 1) & ~15 : s0;
  const size_t head = size_t(2 * a.bt * HD);
  // Where the first of a run's loads finds this lane's 16 bytes, the others by a turn. K: 1024 / RB rows a load, the chunks of row r of the
  // sub-block turned by pi(r); V^T: alike in all of them.
  constexpr int RPL = 1024 / RB, CPR = RB / 16;  // rows of K a load, chunks of a row
  const uint32_t from = kind == 0 ? uint32_t((lane / CPR) * RB + (((lane % CPR) ^ swap23(lane / CPR)) << 4)) : uint32_t((2 * l32 + hb) << 4);
  auto turned = [&](int i) { return kind == 0 ? from ^ uint32_t(swap23(RPL * i) << 4) : from; };
  const uint32_t dst = lds_base + wave * L::kRun;
  // Where this wavefront's next sub-block lies; a stage further is 32 tokens further, past the range the last sub-block again.
  int next_key = n_st > 0 ? min(s0 + 16 * (wave & 1), last_sub) : 0, next_at = next_key / a.bt, next_t0 = next_key - next_at * a.bt;
  if (a.ring) next_at %= a.ring;
  using const_i32 = const int32_t __attribute__((address_space(4)));
  const const_i32* const list = (const const_i32*)a.blocks;
  auto block_id = [&] { return a.ring ? table + next_at : list[table + next_at]; };
  const char* const plane = reinterpret_cast<const char*>(a.pool + size_t(a.kv_base) + size_t(kvh) * head + (kind == 0 ? 0 : size_t(a.bt) * HD));
  const uint64_t block_bytes = uint64_t(a.Hkv) * head * 2;
  const char* next_from = nullptr;  // the run of the stage to be requested next
  auto locate = [&](int id) {
    // (t0 is a multiple of 16: a V^T sub-block starts as far behind its plane as the K row of its first token does)
    next_from = plane + uint64_t(uint32_t(id)) * block_bytes + uint32_t(next_t0 * (HD * 2));
  };
  auto request = [&](int h) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; i += 4)
      load_to_lds16_x4(next_from + 1024 * i, turned(i), turned(i + 1), turned(i + 2), turned(i + 3), dst + uint32_t(h & (kRing - 1)) * L::kStage + 1024 * i);
  };
  auto advance = [&] {
    if (next_key + 32 <= last_sub) {
      next_key += 32;
      next_t0 += 32;
      while (next_t0 >= a.bt) {
        next_t0 -= a.bt;
        if (++next_at == a.ring) next_at = 0;  // (0 on a layer without rings, which it never is again)
      }
    }
  };
  using lds_u32x4 = const __attribute__((address_space(3))) u32x4;
  auto lds_read = [&](uint32_t at) { return *reinterpret_cast<lds_u32x4*>(at); };
  const int prow = swap23(l32);  // the lane with S^T row l32 reads this key of the stage
  const uint32_t k_at = lds_base + (prow >> 4) * L::kRun + (prow & 15) * RB + ((hb ^ (l32 & 15)) << 4);  // its chunk 2 ks + hb: this ^ (ks << 5)
  const uint32_t v_at = lds_base + 2 * L::kRun + lane * 16;

  f32x16 acc[NT];
  float m_ref = -INFINITY, l_run = 0.0f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt] = f32x16{};
  u32x4 P[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};

  f32x16 s{};
  // Matrix work of a stage: P . V of stage h - 1 and the scores of stage h, turn by turn, so that neither waits for its own last result;
  // operands are read two ahead.
  auto products = [&](int h, int next) __attribute__((always_inline)) {
    u32x4 v[3], k[3];
    const uint32_t ka = k_at + uint32_t(h & (kRing - 1)) * L::kStage;
    const uint32_t va = v_at + uint32_t((h - 1) & (kRing - 1)) * L::kStage;
    auto fetch = [&](int g) {
      k[g % 3] = lds_read(ka ^ uint32_t(g << 5));
      v[g % 3] = lds_read(va + (g / NT) * L::kRun + (g % NT) * 1024);
    };
    s = f32x16{};
    fetch(0);
    fetch(1);
#pragma unroll
    for (int g = 0; g < KS; ++g) {
      if (g + 2 < KS) fetch(g + 2);
      s = mfma32x16<DT>(k[g % 3], qf[g], s);
      acc[g % NT] = mfma32x16<DT>(v[g % 3], P[g / NT], acc[g % NT]);
      if (g == KS / 2 - 1 && next >= 0) request(next);
      if (g == KS / 2 && next >= 0) advance();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Lane l holds of S^T, at index 8 sb + i, key 16 sb + 8 hb + i of the stage.
  auto in_range = [&](int k0) {  // the bits of two keys' values
    return (k0 >= rg.from && k0 < rg.end ? 0xffffu : 0u) | (k0 + 1 >= rg.from && k0 + 1 < rg.end ? 0xffff0000u : 0u);
  };
  // Values of a stage with keys that some row does not see, by the wavefront that has staged them: those outside the range may be
  // memory never written, and infinite values of keys that only other rows see must not meet a zero weight. Both become zeros; where
  // there were any of the latter, `bad` says so and marks() keeps which of this lane's outputs they reach: bit e of a word for index e
  // of 32 dims, bit 16 + e for negative ones. They are added at the end.
  int* const bad = reinterpret_cast<int*>(lds + L::kBad);  // [stage of the ring][staging wavefront of the two]
  auto here = [](int x) {  // (what rare code works out from the lane's number is worked out there, not kept through the loop)
    asm volatile("" : "+v"(x));
    return x;
  };
  auto mend = [&](int h) __attribute__((always_inline)) {
    uint32_t found = 0;
    const int ln = here(lane), key0 = s0 + 32 * h + 16 * (wave & 1) + 8 * (ln >> 5);
    char* const mine_at = lds + (uint32_t(h) & (kRing - 1)) * L::kStage + wave * L::kRun + ln * 16;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      u32x4 v = *reinterpret_cast<const u32x4*>(mine_at + i * 1024);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] &= in_range(key0 + 2 * e);
        const uint32_t nf = not_finite2<DT>(v[e]);
        found |= nf;
        v[e] &= ~nf;
      }
      *reinterpret_cast<u32x4*>(mine_at + i * 1024) = v;
    }
    const bool any = __any(found != 0);
    if (ln == 0) bad[2 * (uint32_t(h) & (kRing - 1)) + (wave & 1)] = any;
  };
  bool marked = false;
  auto marks = [&](int h) {
    const int ln = here(lane);
#pragma unroll 1
    for (int w = 0; w < NT; ++w) {
      uint32_t* const word = reinterpret_cast<uint32_t*>(lds + L::kMarks) + (wave * NT + w) * 64 + ln;
      uint32_t found = marked ? *word : 0u;
#pragma unroll 1
      for (int t = 0; t < 32; ++t) {
        const int key = s0 + 32 * h + t;
        if (key < rg.from || key >= rg.end) continue;
        // The row's weight of the key: element t % 8 of P[t / 16], in the lane half (t / 8) % 2.
        uint32_t p2 = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) p2 = i == 4 * (t >> 4) + ((t >> 1) & 3) ? P[i >> 2][i & 3] : p2;
        const float p = __shfl((t & 1) ? unpack_hi<DT>(p2) : unpack_lo<DT>(p2), 32 * ((t >> 3) & 1) + (ln & 31));
        const uint16_t* v = a.pool + size_t(a.kv_base) + (size_t(shaped_block(a, table, key / a.bt)) * size_t(a.Hkv) + size_t(kvh)) * head +
                            vt_elem(a.bt, HD, key % a.bt, 32 * w + 4 * (ln >> 5));
#pragma unroll 1
        for (int e = 0; e < 16; ++e) {
          const uint32_t x = v[(8 * (e >> 2) + (e & 3)) * kVtDim];
          if (!(p > 0.0f)) continue;
          found |= (not_finite_marks<DT>(x, false) & 0xffffu ? 1u << e : 0u) | (not_finite_marks<DT>(x, true) & 0xffffu ? 0x10000u << e : 0u);
        }
      }
      *word = found;
    }
    marked = true;
  };

  constexpr int kAhead = 2;  // stages requested in front of the one at work
  locate(block_id());
  for (int h = 0; h < min(n_st, kAhead); ++h) {
    request(h);
    advance();
    locate(block_id());
  }
  // Q is waited for here, not at its first use in the loop: that wait would be on the counter of the stages on their way.
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
  auto softmax = [&](int h) __attribute__((always_inline)) {
    const float ago = float(s0 + 32 * h + 8 * hb - qpos);
#pragma unroll
    for (int e = 0; e < 16; ++e) s[e] = shaped_score<CAP>(a, s[e]) - slope * fabsf(ago + float(16 * (e >> 3) + (e & 7)));
    if (uint32_t(h - f0) >= uint32_t(f1 - f0)) {
      // The row sees the keys [from, from + n); index e of this lane's half is key 16 (e / 8) + e % 8 behind the first.
      const int lo = max(rg.from, sight.from), n = max(0, min(rg.end, sight.end) - lo);
      const int at = s0 + 32 * h + 8 * (here(lane) >> 5) - lo;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = uint32_t(at + 16 * (e >> 3) + (e & 7)) < uint32_t(n) ? s[e] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = max_halves(mx);
    const bool up = mx > m_ref + kSlack;  // from -inf on: the first key that the row sees
    if (__builtin_expect(__any(up), 0)) {
      const float c = up ? fast_exp2(m_ref - mx) : 1.0f;
      const bool first = m_ref == -INFINITY;
      m_ref = up ? mx : m_ref;
      l_run *= c;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mfma_settle(acc[nt]);
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[nt][e] = first ? 0.0f : acc[nt][e] * c;
      }
    }
    const float off = m_ref == -INFINITY ? 0.0f : m_ref;
    float lx = 0.0f;
#pragma unroll
    for (int sb = 0; sb < 2; ++sb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = 8 * sb + 2 * e;
        const float p0 = fast_exp2(s[at] - off), p1 = fast_exp2(s[at + 1] - off);
        P[sb][e] = pack2<DT>(p0, p1);
        (sb ? lx : l_run) += p0 + p1;
      }
    l_run += lx;
  };
  auto within = [](int h, int lo, int hi) { return uint32_t(h - lo) < uint32_t(hi - lo); };  // (lo <= hi)
  for (int h = 0; h <= n_st; ++h) {
    // All but the stage requested behind this one have landed for this wavefront.
    if (h + 1 < n_st) {
      if constexpr (LOADS == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    if (kind == 1 && h < n_st && !within(h, w0, w1)) {
      mend(h);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    // Behind barrier h stage h has landed for everybody, and nobody reads K of stage h - 1 or V of stage h - 2 any more, whose place in
    // the ring the request takes. On a wavefront's first stage P is zero and the V of "the stage before" whatever lies there, infinities and
    // NaN among it: what that makes of the accumulators goes when a row's reference is first set. On its last turn the scores are not used.
    const bool do_pv = within(h - 1, v0, v1), next_do = h + kAhead < n_st;
    if (do_pv || within(h, v0, v1)) {
      products(h, next_do ? h + kAhead : -1);
    } else if (next_do) {
      request(h + kAhead);
      advance();
    }
    const int id = block_id();
    if (do_pv && !within(h - 1, w0, w1)) {
      const int* b = bad + 2 * ((h - 1) & (kRing - 1));
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(b[0] | b[1]), 0)) marks(h - 1);
    }
    if (within(h, v0, v1)) {
      mfma_settle(s);
      softmax(h);
    }
    locate(id);
  }

  // ---- the rows' end
  const int ln = here(lane), half = ln >> 5;
  const float l = l_run + __shfl_xor(l_run, 32);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) mfma_settle(acc[nt]);
  if (__builtin_expect(marked, 0)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t word = reinterpret_cast<const uint32_t*>(lds + L::kMarks)[(wave * NT + nt) * 64 + ln];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[nt][e] += word >> e & 1 ? INFINITY : 0.0f;
        acc[nt][e] -= word >> (16 + e) & 1 ? INFINITY : 0.0f;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  const bool none = l == 0.0f;  // a row that has seen nothing
  const int col = col0 + (ln & 31);
  const bool live = col < cols_live;
  if (tile.part >= 0) {  // partial records
    if (!live) return;
    const size_t rec = (size_t(tile.part) * a.Hkv + kvh) * a.cols + col;
    float* const to = a.parts_o + rec * HD + 4 * half;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(to + 32 * nt + 8 * i) =
            none ? f32x4{0, 0, 0, 0} : f32x4{acc[nt][4 * i], acc[nt][4 * i + 1], acc[nt][4 * i + 2], acc[nt][4 * i + 3]};
    if (half == 0) {
      a.parts_ml[rec * 2] = m_ref;
      a.parts_ml[rec * 2 + 1] = l;
    }
    return;
  }
  __syncthreads();  // the ring is free
  const float inv = shaped_inverse(l);
  char* const ob = lds + wave * (32 * RB);
  const Place pl = place(ln);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = none ? 0.0f : inv;
      auto x = [&](int j) { return none ? 0.0f : acc[nt][4 * i + j] * f; };
      *reinterpret_cast<u32x2*>(RowsOut<RB>::at(ob, ln & 31, 4 * nt + i) + 8 * half) = u32x2{pack2<DT>(x(0), x(1)), pack2<DT>(x(2), x(3))};
    }
  RowsOut<RB>::store(ob, live ? uint64_t(uintptr_t(a.O + size_t(tile.r0 + pl.m) * a.q_ld + size_t(kvh * a.G + pl.hg) * HD)) : 0, ln);
}

namespace {

template <int DT, int HD>
hipError_t allow_tiled() {
  const hipError_t e = allow_dynamic_lds<attn_shaped_tiled_kernel<DT, HD, false>>(TiledLds<HD>::kBytes);
  return e == hipSuccess ? allow_dynamic_lds<attn_shaped_tiled_kernel<DT, HD, true>>(TiledLds<HD>::kBytes) : e;
}

template <int DT, int HD, bool CAP>
hipError_t launch_tiled_c(const ShapedArgs& a, int n_tiles, hipStream_t st) {
  constexpr auto k = attn_shaped_tiled_kernel<DT, HD, CAP>;
  const hipError_t e = allow_dynamic_lds<k>(TiledLds<HD>::kBytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k, dim3(unsigned(a.Hkv), unsigned(n_tiles)), dim3(256), size_t(TiledLds<HD>::kBytes), st, a);
  return hipGetLastError();
}

template <int DT, int HD>
hipError_t launch_tiled_t(const ShapedArgs& a, int n_tiles, hipStream_t st) {
  return a.cap_log2 > 0.0f ? launch_tiled_c<DT, HD, true>(a, n_tiles, st) : launch_tiled_c<DT, HD, false>(a, n_tiles, st);
}

}  // namespace

hipError_t shaped_tiled_init_attributes() {
  hipError_t e = allow_tiled<ESP_F16, 128>();
  if (e == hipSuccess) e = allow_tiled<ESP_BF16, 128>();
  if (e == hipSuccess) e = allow_tiled<ESP_F16, 256>();
  if (e == hipSuccess) e = allow_tiled<ESP_BF16, 256>();
  return e;
}

// a.cols <= 128 and n_tiles <= 65535: the caller has checked.
hipError_t launch_shaped_tiled(int dt, int HD, const ShapedArgs& a, int n_tiles, hipStream_t st) {
  if (HD == 256) return dt == ESP_F16 ? launch_tiled_t<ESP_F16, 256>(a, n_tiles, st) : launch_tiled_t<ESP_BF16, 256>(a, n_tiles, st);
  return dt == ESP_F16 ? launch_tiled_t<ESP_F16, 128>(a, n_tiles, st) : launch_tiled_t<ESP_BF16, 128>(a, n_tiles, st);
}

}  // namespace esp
