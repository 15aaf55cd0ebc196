// Differential attention (attn_diff.hip says what it computes) for passes with many rows: prompts, chunks, wide drafts.
//
// Bound by the matrix cores: 1536 operations for every pair of query heads, row and visible key. One workgroup is one tile and one KV
// pair; the tile's rows times the G query pairs of the KV pair are up to 128 packed rows (row in tile * G + query pair), so that
// K and V are staged once for all of them and a causal tile's rows lie close together. 8 wavefronts, two for each 32 packed rows, one a
// map. Per 32 keys it computes
//   S^T[32 keys][32 rows] = K_map . Q_map^T      A = K from LDS, B = Q^T in registers
//   P^T = exp2(S^T - m)                          registers; the D layout of S^T is the B layout of P^T
//   O^T[256][32 rows]    += V^T . P^T            A = V^T from LDS, both maps read the same values
// with v_mfma_f32_32x32x16 and P . V one stage behind S. The product takes P in the storage type, as the sum of two such numbers, 16 bits
// or more: 40 products of 32 cycles a stage. So the output's error against 64 bits is that of its own rounding (bf16 0.0017, fp16 0.00021
// of its size), also where the two maps are nearly alike and most of them goes in the difference. One number for both maps: 0.0026 and
// 0.00031, the two cases below in 800 and 48 us. Two for the first and one for the second: 0.0019 and 0.00024 for maps that have nothing in
// common, in 990 and 52 us, but 0.0064 for equal ones at weight 0.8 and 0.029 at 0.95, since what the second loses is not lost by the first
// too. After the last key the second map's wavefronts hand their output over through LDS, and the first map's take the difference, the norm and
// the one rounding of the output.
//
// LDS: a ring of 4 stages of 32 keys, 32 KB each: K of both heads, V^T of both heads, loaded straight from the pool (global_load_lds)
// by wavefronts 0 .. 3 (K, three stages ahead) and 4 .. 7 (V^T, two ahead), a run of 4 KB each. K: the 16-byte chunk c of row r lies at
// c ^ (pi(r) & 15), pi swapping bits 2 and 3; V^T: per sub-block of 16 keys and group of 32 dims [half of the keys][32 dims][8 keys], the
// order in which the lanes of a P . V operand read it. Neither side has bank conflicts. A SIMD has one wavefront of either group; they
// run half a turn apart, so that one's softmax lies under the other's products, and meet at one barrier a turn. Nothing in the loop may
// load from memory but the stages (any such load's wait is a wait for them), nor spill.
//
// 2048 rows behind 12000 keys, 40 / 8 heads, bf16: 1110 to 1150 us, 0.71 to 0.74 PFLOP/s of visible work and 1.19 to 1.23 with the second
// numbers, where a plain 8192^3 product of the library reaches 1.20. A SIMD's matrix core is busy 75 % of the time that a workgroup is there (other vector
// work beside it for 43 % of that), and one is there 83 % of the pass. Ragged fresh prompts of 40 .. 800 rows, 32 / 8, fp16: 56 to 57 us, the
// longest tile's 25 stages and the turns before and after them, in which the matrix cores are busy 45 %.
#include "diff_math.hpp"
#include "lds_direct.hpp"

namespace esp {

namespace {
constexpr int kRing = 4, kStage = 32 * 1024;  // stages; bytes of one
constexpr int kOffBad = kRing * kStage, kOffMarks = kOffBad + 64;     // 16 ints behind the ring; then a word per lane and 32 dims
constexpr size_t kDiffTiledLds = kOffMarks + 8 * (kDiffVD / 32) * 256;
constexpr float kSlack = 8.0f;  // a row's reference moves when a score exceeds it by more (log2 units): P stays below 2^8

// The maximum over the two lanes that hold a row. (Of the builtin for this instruction the compiler keeps one result only; the two
// wait states are what it puts between a vector instruction and the exchange of its result.)
__device__ __forceinline__ float max_halves(float x) {
  float y = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}
}  // namespace

template <int DT>
__global__ __launch_bounds__(512, 2) void attn_diff_tiled_kernel(const DiffArgs a) {
  constexpr int HD = kDiffHD, VD = kDiffVD, NT = VD / 32, KS = HD / 16;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const uint32_t lds_base = uint32_t(uintptr_t(lds));
  const int j = blockIdx.x;  // KV pair
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l32 = lane & 31, hb = lane >> 5, map = (wave ^ (wave >> 2)) & 1, col0 = 32 * (wave >> 1);
  const esp_tile tile = a.tiles[gridDim.y - 1 - blockIdx.y];  // last to first: a causal pass's longest tiles start first
  const esp_tree tree = a.trees[tile.tree];
  const int table = tile.pad > 0 ? tile.pad - 1 : tree.table;
  const DiffRange rg = diff_range(tile, tree, a.R, a.window);
  const int cols_live = rg.rows * a.G;

  // ---- this lane's packed row
  struct Place {
    int m, hg;  // row in the tile, query pair of the KV pair; row 0's first where there is none
  };
  auto place = [&](int l) {
    const int col = col0 + (l & 31);
    const bool ok = col < cols_live;
    const int m = ok ? col / a.G : 0;
    return Place{m, ok ? col - m * a.G : 0};
  };
  u32x4 qf[KS];
  int qpos;
  {
    const Place pl = place(lane);
    qpos = tree.P + rg.rr0 + pl.m;
    const uint16_t* qp = a.Q + size_t(tile.r0 + pl.m) * a.q_ld + size_t(2 * (j * a.G + pl.hg) + map) * HD + 8 * hb;
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
  // Where the first of a run's four loads finds this lane's 16 bytes. K: four rows a load, the chunks of row r of the sub-block turned by
  // pi(r), so those of the other loads differ by pi(4 i); V^T: alike in all of them.
  const uint32_t from = kind < 2 ? uint32_t((lane >> 4) * 256 + (((lane & 15) ^ swap23(lane >> 4)) << 4)) : uint32_t((2 * l32 + hb) << 4);
  const uint32_t turn1 = kind < 2 ? swap23(4) << 4 : 0, turn2 = kind < 2 ? swap23(8) << 4 : 0;
  const uint32_t dst = lds_base + wave * 4096;
  // Where this wavefront's next sub-block lies; a stage further is 32 tokens further, past the range the last sub-block again.
  int next_key = n_st > 0 ? min(s0 + 16 * (wave & 1), last_sub) : 0, next_at = next_key / a.bt, next_t0 = next_key - next_at * a.bt;
  if (a.ring) next_at %= a.ring;
  using const_i32 = const int32_t __attribute__((address_space(4)));
  const const_i32* const list = (const const_i32*)a.blocks;
  auto block_id = [&] { return a.ring ? table + next_at : list[table + next_at]; };
  const char* const plane = reinterpret_cast<const char*>(a.pool + size_t(a.kv_base) + size_t(2 * j + (kind & 1)) * head + (kind < 2 ? 0 : size_t(a.bt) * HD));
  const uint64_t block_bytes = uint64_t(a.Hkv) * head * 2;
  const char* next_from = nullptr;  // the run of the stage to be requested next
  auto locate = [&](int id) {
    // (t0 is a multiple of 16: a V^T sub-block starts as far behind its plane as the K row of its first token does)
    next_from = plane + uint64_t(uint32_t(id)) * block_bytes + uint32_t(next_t0 * (HD * 2));
  };
  auto request = [&](int h) __attribute__((always_inline)) {
    load_to_lds16_x4(next_from, from, from ^ turn1, from ^ turn2, from ^ turn1 ^ turn2, dst + uint32_t(h & (kRing - 1)) * kStage);
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
  // Runs in a stage: K of head 0 sub-block 0, 1, K of head 1, V^T of head 0, V^T of head 1; 4 KB each.
  using lds_u32x4 = const __attribute__((address_space(3))) u32x4;
  auto lds_read = [&](uint32_t at) { return *reinterpret_cast<lds_u32x4*>(at); };
  const int prow = swap23(l32);  // the lane with S^T row l32 reads this key of the stage
  const uint32_t k_at = lds_base + map * 8192 + prow * 256 + ((hb ^ (l32 & 15)) << 4);  // its chunk 2 ks + hb: this ^ (ks << 5)
  const uint32_t v_at = lds_base + 16384 + lane * 16;

  f32x16 acc[NT];
  float m_ref = -INFINITY, l_run = 0.0f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) acc[nt] = f32x16{};
  u32x4 P[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}}, rest[2] = {u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};  // rest: what P's rounding left

  f32x16 s{};
  // Matrix work of a turn, and the request of stage `next` (-1: none) between it: P . V of stage h - 1 and the scores of stage h, a score
  // product in front of every two of P . V so that neither waits for its own last result; operands are read two groups of three ahead.
  auto products = [&](int h, int next) __attribute__((always_inline)) {
    u32x4 v[3][2], k[3];
    const uint32_t ka = k_at + uint32_t(h & (kRing - 1)) * kStage;
    uint32_t va = v_at + uint32_t((h - 1) & (kRing - 1)) * kStage;
    asm("" : "+v"(va));  // one register, the operands' places as immediates: left alone the compiler keeps eight
    auto fetch = [&](int g) {
      k[g % 3] = lds_read(ka ^ uint32_t(g << 5));
#pragma unroll
      for (int i = 0; i < 2; ++i) v[g % 3][i] = lds_read(va + ((2 * g + i) >> 2 & 1) * 8192 + ((2 * g + i) >> 3) * 4096 + ((2 * g + i) & 3) * 1024);
    };
    s = f32x16{};
    fetch(0);
    fetch(1);
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      if (g < 6) fetch(g + 2);
      s = mfma32x16<DT>(k[g % 3], qf[g], s);
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[(2 * g + i) & 7] = mfma32x16<DT>(v[g % 3][i], P[g >> 2], acc[(2 * g + i) & 7]);
#pragma unroll
      for (int i = 0; i < 2; ++i) acc[(2 * g + i) & 7] = mfma32x16<DT>(v[g % 3][i], rest[g >> 2], acc[(2 * g + i) & 7]);
      if (g == 3 && next >= 0) request(next);
      if (g == 5 && next >= 0) advance();
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Lane l holds of S^T, at index 8 sb + i, key 16 sb + 8 hb + i of the stage.
  auto in_range = [&](int k0) {  // the bits of two keys' values
    return (k0 >= rg.lo && k0 < rg.hi ? 0xffffu : 0u) | (k0 + 1 >= rg.lo && k0 + 1 < rg.hi ? 0xffff0000u : 0u);
  };
  // Values of a stage with keys that some row does not see, by the wavefront that has staged them: those outside the range may be
  // memory never written, and infinite values of keys that only other rows see must not meet a zero weight. Both become zeros; where
  // there were any of the latter, `bad` says so and marks() keeps which of this lane's outputs they reach: bit e of a word for index e
  // of 32 dims, bit 16 + e for negative ones. They are added at the end (a branch of the loop that touched the accumulators would cost
  // registers in every turn).
  int* const bad = reinterpret_cast<int*>(lds + kOffBad);  // [stage of the ring][staging wavefront of the four]
  // (What such rare code works out from the lane's number is worked out there: kept in registers through the loop it would cost spills.)
  auto here = [](int x) {
    asm volatile("" : "+v"(x));
    return x;
  };
  auto mend = [&](int h) __attribute__((always_inline)) {
    uint32_t found = 0;
    const int ln = here(lane), key0 = s0 + 32 * h + 16 * (wave & 1) + 8 * (ln >> 5);
    char* const mine = lds + (uint32_t(h) & (kRing - 1)) * kStage + wave * 4096 + ln * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 v = *reinterpret_cast<const u32x4*>(mine + i * 1024);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] &= in_range(key0 + 2 * e);
        const uint32_t nf = not_finite2<DT>(v[e]);
        found |= nf;
        v[e] &= ~nf;
      }
      *reinterpret_cast<u32x4*>(mine + i * 1024) = v;
    }
    const bool any = __any(found != 0);
    if (ln == 0) bad[4 * (uint32_t(h) & (kRing - 1)) + (wave & 3)] = any;
  };
  bool marked = false;
  auto marks = [&](int h) {
    const int ln = here(lane);
#pragma unroll 1
    for (int w = 0; w < NT; ++w) {
      uint32_t* const word = reinterpret_cast<uint32_t*>(lds + kOffMarks) + (wave * NT + w) * 64 + ln;
      uint32_t found = marked ? *word : 0u;
#pragma unroll 1
      for (int t = 0; t < 32; ++t) {
        const int key = s0 + 32 * h + t;
        if (key < rg.lo || key >= rg.hi) continue;
        // The row's weight of the key: element t % 8 of P[t / 16], in the lane half (t / 8) % 2.
        uint32_t p2 = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) p2 = i == 4 * (t >> 4) + ((t >> 1) & 3) ? P[i >> 2][i & 3] : p2;
        const float p = __shfl((t & 1) ? unpack_hi<DT>(p2) : unpack_lo<DT>(p2), 32 * ((t >> 3) & 1) + (ln & 31));
        const uint16_t* v = a.pool + diff_head_base(a, diff_block(a, table, key / a.bt), 2 * j + (w >> 2)) +
                            vt_elem(a.bt, HD, key % a.bt, 32 * (w & 3) + 4 * (ln >> 5));
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

  const bool late = wave >= 4;
  const int ahead = late ? 2 : 3;  // how many stages ahead of its matrix work a wavefront requests
  locate(block_id());
  for (int h = 0; h < min(n_st, ahead); ++h) {
    request(h);
    advance();
    locate(block_id());
  }
  // Q is waited for here, not at its first use in the loop: that wait would be on the counter of the stages on their way.
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
  auto meet = [&] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto wait_behind = [&](int n) {  // all but the last n stages requested have landed for this wavefront, 4 loads each
    if (n >= 2) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else if (n == 1) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  };
  auto softmax = [&]() __attribute__((always_inline)) {
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    mx = max_halves(mx) * a.scale_log2;
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
        const float p0 = fast_exp2(s[at] * a.scale_log2 - off), p1 = fast_exp2(s[at + 1] * a.scale_log2 - off);
        P[sb][e] = pack2<DT>(p0, p1);
        rest[sb][e] = pack2<DT>(p0 - unpack_lo<DT>(P[sb][e]), p1 - unpack_hi<DT>(P[sb][e]));
        (sb ? lx : l_run) += p0 + p1;
      }
    l_run += lx;
  };
  // The two groups of wavefronts, one wavefront of each on a SIMD: the early one (0 .. 3, which stage K) and the late one (4 .. 7, which
  // stage V). One barrier a turn: the early group passes it in front of its matrix work, the late one in front of its softmax, so that
  // while one has its matrix work the other has its softmax. Behind barrier h, K of stage h and V of stage h - 1 have landed for
  // everybody, and nobody reads K of stage h - 1 (whose place the early group's next request takes) or V of stage h - 2 (the late one's) any more.
  auto within = [](int h, int lo, int hi) { return uint32_t(h - lo) < uint32_t(hi - lo); };  // (lo <= hi)
  if (late) meet();
  for (int h = 0; h <= n_st; ++h) {
    if (!late) {
      wait_behind(n_st - 1 - h);  // K of stage h: up to two stages requested behind it
      meet();
    }
    // On a wavefront's first stage P is zero and the V of "the stage before" whatever lies there, infinities and NaN among it: what that
    // makes of the accumulators goes when a row's reference is first set. On its last turn the scores are not used.
    const bool do_pv = within(h - 1, v0, v1);
    const int next = h + ahead < n_st ? h + ahead : -1;
    if (do_pv || within(h, v0, v1)) {
      __builtin_amdgcn_s_setprio(1);
      products(h, next);
      __builtin_amdgcn_s_setprio(0);
    } else if (next >= 0) {
      request(next);
      advance();
    }
    if (late) {
      wait_behind(n_st - 1 - h);  // V of stage h
      if (h < n_st && !within(h, w0, w1)) {
        mend(h);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      meet();
    }
    const int id = block_id();
    if (do_pv && !within(h - 1, w0, w1)) {
      const int* b = bad + 4 * ((h - 1) & (kRing - 1));
      if (__builtin_expect(__builtin_amdgcn_readfirstlane(b[0] | b[1] | b[2] | b[3]), 0)) marks(h - 1);
    }
    if (within(h, v0, v1)) {
      if (!within(h, f0, f1)) {
        mfma_settle(s);
        // The row sees the keys [from, from + n); index e of this lane's half is key 16 (e / 8) + e % 8 behind the first.
        const int from = a.window > 0 ? max(rg.lo, qpos - a.window + 1) : rg.lo, n = max(0, min(rg.hi, qpos + 1) - from);
        const int at = s0 + 32 * h + 8 * (here(lane) >> 5) - from;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = uint32_t(at + 16 * (e >> 3) + (e & 7)) < uint32_t(n) ? s[e] : -INFINITY;
      }
      softmax();
    }
    locate(id);
  }
  if (!late) meet();

  // ---- the rows' end. 32 packed rows of 256 fp32 numbers pass through 32 KB of the ring, the two wavefronts of the rows' maps on each
  // side: written by a lane for its row (4 dims at a time: g = 0 .. 31, its half's of dims 8 g .. 8 g + 7), read a row by 32 lanes, 8 dims
  // each, so that rows leave in whole lines. Lane by lane from the accumulators they left 8 bytes at a time: 8 us of a workgroup's time.
  const int ln = here(lane), half = ln >> 5, l5 = ln & 31;
  float l = l_run + __shfl_xor(l_run, 32);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) mfma_settle(acc[nt]);
  if (__builtin_expect(marked, 0)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint32_t word = reinterpret_cast<const uint32_t*>(lds + kOffMarks)[(wave * NT + nt) * 64 + ln];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        acc[nt][e] += word >> e & 1 ? INFINITY : 0.0f;
        acc[nt][e] -= word >> (16 + e) & 1 ? INFINITY : 0.0f;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  const bool none = l == 0.0f;  // a row that has seen nothing
  if (__any(none)) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[nt][e] = none ? 0.0f : acc[nt][e];
  }
  // 4 dims of a row: at 1 KB * g + 512 * half + 16 * (row ^ g), turned by g: no bank conflicts on either side. The lane's own are at
  // mine() ^ 16 g + 1 KB * g, its part asked for anew by each pass over them: 32 addresses kept for the next pass would be spilled.
  char* const rows = lds + (wave >> 1) * 32768;
  auto mine = [&] {
    const int x = here(lane);
    return 512 * (x >> 5) + 16 * (x & 31);
  };
  auto own = [&](int at, int g) { return reinterpret_cast<f32x4*>(rows + (at ^ (16 * g)) + 1024 * g); };
  auto put = [&](float f) __attribute__((always_inline)) {
    const int at = mine();
#pragma unroll
    for (int g = 0; g < 32; ++g)
      *own(at, g) = f32x4{acc[g >> 2][4 * (g & 3)] * f, acc[g >> 2][4 * (g & 3) + 1] * f, acc[g >> 2][4 * (g & 3) + 2] * f, acc[g >> 2][4 * (g & 3) + 3] * f};
  };
  // The wavefront's half of the rows, two at a time: take(packed row, its dims 8 l5 .. + 3, + 4 .. + 7).
  auto leave = [&](auto take) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const int row = 16 * map + 2 * i + half;
      const char* const at = rows + 1024 * l5 + 16 * (row ^ l5);
      if (col0 + row < cols_live) take(col0 + row, *reinterpret_cast<const f32x4*>(at), *reinterpret_cast<const f32x4*>(at + 512));
    }
  };
  __syncthreads();  // the ring is free
  if (tile.part >= 0) {  // partial records
    float* const to = a.parts_o + (size_t(tile.part) * (a.Hkv / 2) + j) * 2 * a.cols * VD + 8 * l5;
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
      if (map == e) put(1.0f);
      __syncthreads();
      leave([&](int col, f32x4 x, f32x4 y) {
        f32x4* const rec = reinterpret_cast<f32x4*>(to + (size_t(e) * a.cols + col) * VD);
        rec[0] = x;
        rec[1] = y;
      });
      __syncthreads();
    }
    if (half == 0 && col0 + l5 < cols_live) {
      float* const ml = a.parts_ml + (((size_t(tile.part) * (a.Hkv / 2) + j) * 2 + map) * a.cols + col0 + l5) * 2;
      ml[0] = m_ref;
      ml[1] = l;
    }
    return;
  }
  if (map == 1) put(diff_inverse(l) * a.weight[j * a.G + place(ln).hg]);
  __syncthreads();
  float* const factors = reinterpret_cast<float*>(lds + kOffMarks) + col0;  // the norm's of every packed row
  if (map == 0) {
    const float f1 = diff_inverse(l);
    float ss = 0.0f;
    const int at = mine();
#pragma unroll
    for (int g = 0; g < 32; ++g) {
      f32x4* const x = own(at, g);
      f32x4 o = f32x4{acc[g >> 2][4 * (g & 3)], acc[g >> 2][4 * (g & 3) + 1], acc[g >> 2][4 * (g & 3) + 2], acc[g >> 2][4 * (g & 3) + 3]} * f1 - *x;
      *x = o;
      ss += o[0] * o[0] + o[1] * o[1] + o[2] * o[2] + o[3] * o[3];
    }
    ss += __shfl_xor(ss, 32);
    if (half == 0) factors[l5] = a.norm_w ? a.factor * rsqrtf(ss * (1.0f / VD) + a.eps) : a.factor;
  }
  f32x4 w[2] = {{1, 1, 1, 1}, {1, 1, 1, 1}};
  if (a.norm_w) {
    w[0] = *reinterpret_cast<const f32x4*>(a.norm_w + 8 * l5);
    w[1] = *reinterpret_cast<const f32x4*>(a.norm_w + 8 * l5 + 4);
  }
  __syncthreads();
  leave([&](int col, f32x4 x, f32x4 y) {
    const float f = factors[col - col0];
    x *= w[0] * f;
    y *= w[1] * f;
    const int m = col / a.G;
    using out16 = uint32_t __attribute__((ext_vector_type(4), aligned(8)));  // a row of O starts at any multiple of 8 bytes
    *reinterpret_cast<out16*>(a.O + size_t(tile.r0 + m) * a.q_ld + size_t(j * a.G + col - m * a.G) * VD + 8 * l5) =
        out16{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]), pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
  });
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
