// Attention with shaped scores (attn_shaped.hip says what it computes) for passes with many rows: prompts, chunks, wide drafts.
//
// Bound by the matrix cores and the vector units beside them: 4 head_dim operations for every query head, row and visible key, and one
// exponential for its weight, two more for a cap. One workgroup is one tile and one KV head; the tile's rows times the G
// query heads are up to 128 packed rows (row in tile * G + head of the group), 32 a wavefront. Per 32 keys a wavefront computes
//   S^T[32 keys][32 rows] = K . Q^T      A = K from LDS, B = Q^T in registers
//   P^T = exp2(shaped(S^T) - m)          registers; the D layout of S^T is the B layout of P^T
//   O^T[head_dim][32 rows] += V^T . P^T  A = V^T from LDS
// with v_mfma_f32_32x32x16. A turn has three stages in hand: the scores of stage h are made under the caps of stage h - 1's (without a cap: under
// half of its exponentials), P . V of stage h - 2 under the exponentials of stage h - 1, so that matrix and vector units work beside each other
// within a wavefront too. Turns that are not all of that - the ends of a range, masked stages - run the three one by one.
//
// Scores: the bias is what the score product's accumulator starts from (without a cap; behind a cap it is the last step's addend), but for
// what it has of the stage, which is taken from the reference. A cap is tanh as an odd polynomial where all of a wavefront's scores of the
// stage are below 0.2 caps (four operations a score) or 0.7 (six), else by an exponential and a reciprocal (eleven). 2048 rows behind 8000 keys,
// 32 / 8 heads of 128 dims, bf16, 303 billion operations, us: plain 424, with slopes 416, with a cap, with slopes or without, 472 (scores below 0.2
// caps), 494 (0.7) and 505 (above), 0.60 to 0.73 PFLOP/s and half as much again with the weights' second numbers, matrix units busy 47 % and vector
// units 60 % of the clocks; 16 / 8 heads of 256 dims: plain 421, with a cap 462, 473 and 476. Short ranges are bound by their ends: three prompts of
// 500 to 2000 rows in six documents each take 60 to 66 us, of which a tile's seven stages are a third, its first loads from memory another.
//
// P enters its product as the sum of two numbers of the storage type, 16 bits or more, as in the streaming kernel, so that a row is as exact
// in a pass of many rows as in one of few: an output's error is that of its own rounding. One number, half of P . V's matrix work, makes it up to 1.4
// times as much, 0.0023 of the output's size for 0.0017 (bf16): the chunk with both then takes 392 us, the packed documents 52 to 57.
//
// LDS: a ring of 4 stages of 32 keys, K and V^T, loaded straight from the pool (global_load_lds): wavefronts 0 and 1 load the
// two sub-blocks of K, two stages ahead of the scores, 2 and 3 those of V^T, two ahead of P . V. K: the 16-byte chunk c of row r lies at
// c ^ (pi(r) & 15), pi swapping bits 2 and 3; V^T: per sub-block of 16 keys and group of 32 dims [half of the keys][32 dims][8 keys], the
// order in which the lanes of a P . V operand read it. Neither side has bank conflicts. Nothing in the loop may load from memory but the
// stages (any such load's wait is a wait for them).
#include "lds_direct.hpp"
#include "rows_out.hpp"
#include "shaped_math.hpp"

#include <type_traits>

namespace esp {

namespace {
constexpr int kRing = 4;
constexpr float kSlack = 8.0f;  // a row's reference moves when a score exceeds it by more (log2 units): P stays below 2^8
// Of fp16 the reference lies 7 below the score that it is taken from, so that weights go up to 2^15 and a number's last step, 2^-24, is 2^-31 of
// that score's or less. (Not where fp32 does not hold the difference.)
template <int DT>
constexpr float kBelow = DT == ESP_F16 ? 7.0f : 0.0f;
template <int DT>
__device__ __forceinline__ float reference_of(float x) {
  return DT == ESP_F16 && fabsf(x) < 0x1p20f ? x - kBelow<DT> : x;
}
template <int DT>
constexpr float kMost = DT == ESP_F16 ? 0x1p15f : 0x1p8f;  // where slack is not looked for: when a lane's weights of a stage come to more

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

// The largest of a wavefront's numbers (none the lowest there is): over rows of 16 lanes, then from row to row.
template <int CTRL, int ROWS>
__device__ __forceinline__ int most_from(int x) {
  return max(x, __builtin_amdgcn_update_dpp(INT32_MIN, x, CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ int wave_most(int x) {
  x = most_from<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = most_from<0x112, 0xf>(x);
  x = most_from<0x114, 0xf>(x);
  x = most_from<0x118, 0xf>(x);
  x = most_from<0x142, 0xa>(x);  // row_bcast 15, 31
  x = most_from<0x143, 0xc>(x);
  return __builtin_amdgcn_readlane(x, 63);
}

// The order of a block of matrix instructions, M for each of N operands from LDS two ahead: one, then V vector operations (exponentials
// among them), and the operand of the one after the next.
template <int N, int M, int V>
__device__ __forceinline__ void lay_out() {
  __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
  for (int g = 0; g < N; ++g) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, V, 0);
    }
  }
}

// A lane's 16 weights of a stage, two to a dword, as the sum of two numbers of the storage type each.
struct Weights {
  u32x4 p[2], rest[2];
};
template <int DT>
__device__ __forceinline__ void put_weights(Weights& w, int sb, int e, float p0, float p1, float& sum) {
  uint32_t p = pack2<DT>(p0, p1);
  asm("" : "+v"(p));  // (left alone the compiler converts the lower one once more instead of shifting it out)
  w.p[sb][e] = p;
  w.rest[sb][e] = pack2<DT>(p0 - unpack_lo<DT>(p), p1 - unpack_hi<DT>(p));
  sum = sum2<DT>(w.rest[sb][e], sum2<DT>(p, sum));  // (the weights as the product takes them)
}
}  // namespace

template <int DT, int HD, bool CAP, bool BIAS>
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
    // In the units of the score that it is added to: the product's, or behind a cap log2 units.
    slope = BIAS ? a.slopes[kvh * a.G + pl.hg] * (CAP ? kLog2e : kLog2e / a.scale_log2) : 0.0f;
  }
  // What some and what all of a set of rows see: of this wavefront's and of the tile's.
  struct Seen {
    int some_from, some_end, all_from, all_end;
  };
  Seen mine{}, whole{};
  const int q_first = tree.P + rr0 + min(col0, cols_live - 1) / a.G;  // of this wavefront's rows
  if (a.spans) {
    auto reduce = [](const Seen& s) { return Seen{-wave_most(-s.some_from), wave_most(s.some_end), wave_most(s.all_from), -wave_most(-s.all_end)}; };
    mine = reduce(Seen{sight.from, sight.end, sight.from, sight.end});
    const int m0 = min(lane, rows - 1), m1 = min(lane + 64, rows - 1);
    const Sight s0 = shaped_sight(a, tile.r0 + m0, tree.P + rr0 + m0, n_keys), s1 = shaped_sight(a, tile.r0 + m1, tree.P + rr0 + m1, n_keys);
    whole = reduce(Seen{min(s0.from, s1.from), max(s0.end, s1.end), max(s0.from, s1.from), min(s0.end, s1.end)});
  } else {
    auto of_rows = [&](int m0, int m1) {
      const int q0 = tree.P + rr0 + m0, q1 = tree.P + rr0 + m1;
      return Seen{a.window > 0 ? max(0, q0 - a.window + 1) : 0, q1 + 1, a.window > 0 ? max(0, q1 - a.window + 1) : 0, q0 + 1};
    };
    mine = of_rows(min(col0, cols_live - 1) / a.G, (min(col0 + 32, cols_live) - 1) / a.G);
    whole = of_rows(0, rows - 1);
  }
  const Sight rg = shaped_range(tile, tree, whole.some_from, whole.some_end);

  // ---- stages of 32 keys, the last ones first: a bias makes near keys' scores the largest, and taken from the far ones on every stage's would
  // move the reference (2048 rows behind 8000 keys, 32 / 8 heads, 8 of them of slopes above 0.17, with single weights: 500 us for 354). Stage h
  // holds the keys from key_of(h) on, the last stage's from the sub-block of the first key on. Which stages this wavefront's rows see, and which
  // whole:
  const int s0 = rg.from & ~15;
  const int n_st = rg.end > rg.from ? (rg.end - s0 + 31) >> 5 : 0;
  auto key_of = [&](int h) { return s0 + 32 * (n_st - 1 - h); };
  auto turn_round = [&](int& x0, int& x1) {
    const int y = n_st - x1;
    x1 = n_st - x0;
    x0 = y;
  };
  int v0 = 0, v1 = 0, f0 = 0, f1 = 0;  // stages [v0, v1) hold keys that some row sees, [f0, f1) only keys that all see
  int w0 = 0, w1 = 0;                  // [w0, w1) only keys that all rows of the tile see
  if (n_st && col0 < cols_live) {
    const int some_lo = max(rg.from, mine.some_from), some_hi = min(rg.end, mine.some_end);
    const int all_lo = max(rg.from, mine.all_from), all_hi = min(rg.end, mine.all_end);
    if (some_hi > some_lo) {
      v0 = (some_lo - s0) >> 5;
      v1 = (some_hi - s0 + 31) >> 5;
      f0 = (all_lo - s0 + 31) >> 5;
      f1 = max(f0, ((BIAS ? min(all_hi, q_first + 1) : all_hi) - s0) >> 5);  // (behind a row's own key its bias falls again)
    }
  }
  if (n_st) {
    w0 = (max(rg.from, whole.all_from) - s0 + 31) >> 5;
    w1 = max(w0, (min(rg.end, whole.all_end) - s0) >> 5);
    turn_round(w0, w1);
  }
  turn_round(v0, v1);
  turn_round(f0, f1);

  // ---- staging: wavefront w loads sub-block w % 2 of K or V (w / 2) of every stage
  const int kind = wave >> 1, last_sub = rg.end > rg.from ? (rg.end - 1) & ~15 : s0;
  const size_t head = size_t(2 * a.bt * HD);
  // Where the first of a run's loads finds this lane's 16 bytes, the others by a turn. K: 1024 / RB rows a load, the chunks of row r of the
  // sub-block turned by pi(r); V^T: alike in all of them.
  constexpr int RPL = 1024 / RB, CPR = RB / 16;  // rows of K a load, chunks of a row
  const uint32_t from = kind == 0 ? uint32_t((lane / CPR) * RB + (((lane % CPR) ^ swap23(lane / CPR)) << 4)) : uint32_t((2 * l32 + hb) << 4);
  auto turned = [&](int i) { return kind == 0 ? from ^ uint32_t(swap23(RPL * i) << 4) : from; };
  const uint32_t dst = lds_base + wave * L::kRun;
  // Where this wavefront's next sub-block lies; a stage further is 32 tokens further down. Past the range's end the last sub-block again.
  int next_raw, next_key, next_at, next_t0;
  auto start = [&]() __attribute__((always_inline)) {
    next_raw = n_st > 0 ? key_of(0) + 16 * (wave & 1) : 0;
    next_key = min(next_raw, last_sub);
    next_at = next_key / a.bt;
    next_t0 = next_key - next_at * a.bt;
    if (a.ring) next_at %= a.ring;
  };
  using const_i32 = const int32_t __attribute__((address_space(4)));
  const const_i32* const list = (const const_i32*)a.blocks;
  auto block_id = [&] { return a.ring ? table + next_at : list[table + next_at]; };
  const char* const plane = reinterpret_cast<const char*>(a.pool + size_t(a.kv_base) + size_t(kvh) * head + (kind == 0 ? 0 : size_t(a.bt) * HD));
  const uint64_t block_bytes = uint64_t(a.Hkv) * head * 2;
  const char* next_from[2] = {};  // the runs of the two stages to be requested next
  auto locate = [&](int id, int t0) __attribute__((always_inline)) {
    // (t0 is a multiple of 16: a V^T sub-block starts as far behind its plane as the K row of its first token does)
    return plane + uint64_t(uint32_t(id)) * block_bytes + uint32_t(t0 * (HD * 2));
  };
  auto request = [&](int h, int i, int which) __attribute__((always_inline)) {
    load_to_lds16(next_from[which] + 1024 * i, turned(i), dst + uint32_t(h & (kRing - 1)) * L::kStage + 1024 * i);
  };
  auto request_all = [&](int h, int which) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) request(h, i, which);
  };
  auto advance = [&]() __attribute__((always_inline)) {
    if (next_raw - 32 >= s0) {
      next_raw -= 32;
      next_t0 -= next_key - next_raw;
      next_key = next_raw;
      while (next_t0 < 0) {
        next_t0 += a.bt;
        if (--next_at < 0) next_at = a.ring - 1;  // (a layer without rings has no blocks in front of the first key's)
      }
    }
  };
  // The two stages behind those that were located last: their blocks now, where they lie when the scalar loads are there.
  int next_id[2], at_t0[2];
  auto look_up = [&](int which) __attribute__((always_inline)) {
    advance();
    next_id[which] = block_id();
    at_t0[which] = next_t0;
  };
  auto locate_both = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) next_from[i] = locate(next_id[i], at_t0[i]);
  };
  using lds_u32x4 = const __attribute__((address_space(3))) u32x4;
  auto lds_read = [&](uint32_t at) { return *reinterpret_cast<lds_u32x4*>(at); };
  const int prow = swap23(l32);  // the lane with S^T row l32 reads this key of the stage
  const uint32_t k_at = lds_base + (prow >> 4) * L::kRun + (prow & 15) * RB + ((hb ^ (l32 & 15)) << 4);  // its chunk 2 ks + hb: this ^ (ks << 5)
  const uint32_t v_at = lds_base + 2 * L::kRun + lane * 16;

  f32x16 acc[NT];
  float m_ref, l_run;
  // Scores and weights of the stage at work and of the one before, by the stage's parity.
  f32x16 s[2] = {f32x16{}, f32x16{}};
  Weights P[2] = {};

  // The bias of index e of this lane's half, linear in the key: right up to the row's own key. A part for the index, which never changes, and
  // one for the stage, which joins the scores where they are taken from the reference.
  auto bias_at = [&](int h) { return BIAS ? slope * float(key_of(h) + 8 * hb - qpos) : 0.0f; };
  f32x16 bias;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    bias[e] = BIAS ? slope * float(16 * (e >> 3) + (e & 7)) : 0.0f;
    if constexpr (BIAS && HD == 128) asm("" : "+v"(bias[e]));
  }
  auto value_operand = [&](uint32_t va, int g) { return lds_read(va + (g / NT) * L::kRun + (g % NT) * 1024); };
  auto values_of = [&](int h) {
    uint32_t va = v_at + uint32_t(h & (kRing - 1)) * L::kStage;
    asm("" : "+v"(va));  // one register, the operands' places as immediates
    return va;
  };
  // S = K Q^T of stage h (+ the indexes' bias / scale), operands read two ahead; `between` is work to be laid under it.
  auto score = [&](int h, f32x16& to, auto between) __attribute__((always_inline)) {
    u32x4 k[3];
    const uint32_t ka = k_at + uint32_t(h & (kRing - 1)) * L::kStage;
    auto fetch = [&](int g) { k[g % 3] = lds_read(ka ^ uint32_t(g << 5)); };
    fetch(0);
    fetch(1);
#pragma unroll
    for (int g = 0; g < KS; ++g) {
      if (g + 2 < KS) fetch(g + 2);
      to = mfma32x16<DT>(k[g % 3], qf[g], g > 0 ? to : BIAS && !CAP ? bias : f32x16{});
      between(g);
      __builtin_amdgcn_sched_barrier(0x406);  // (vector and scalar work may cross; operands' reads and products keep their order)
    }
  };
  // O^T += V^T P^T of stage h.
  auto weigh = [&](int h, const Weights& w, auto between) __attribute__((always_inline)) {
    u32x4 v[3];
    const uint32_t va = values_of(h);
    auto fetch = [&](int g) { v[g % 3] = value_operand(va, g); };
    fetch(0);
    fetch(1);
#pragma unroll
    for (int g = 0; g < 2 * NT; ++g) {
      if (g + 2 < 2 * NT) fetch(g + 2);
      acc[g % NT] = mfma32x16<DT>(v[g % 3], w.p[g / NT], acc[g % NT]);
      acc[g % NT] = mfma32x16<DT>(v[g % 3], w.rest[g / NT], acc[g % NT]);
      between(g);
      __builtin_amdgcn_sched_barrier(0x406);
    }
  };
  // From products to scores in log2 units (BIAS without a cap: the bias is in already).
  auto largest_size = [&](const f32x16& x) {
    float m = fabsf(x[0]);
#pragma unroll
    for (int e = 1; e < 16; ++e) m = fmaxf(m, fabsf(x[e]));
    return m;
  };
  auto shape_e = [&](float x, int e, auto terms) __attribute__((always_inline)) {  // terms of the polynomial; 0: the exponential
    if constexpr (!CAP) return x;
    else if constexpr (terms == 3) return shaped_tanh_short(a, x, bias[e]);
    else if constexpr (terms == 5) return shaped_tanh_low(a, x, bias[e]);
    else return shaped_tanh_high(a, x, bias[e]);
  };
  // With a cap scores are in log2 units, else still in those of the products.
  const float unit = CAP ? 1.0f : a.scale_log2;
  // `far`: for rows whose reference is in the millions or more, where fp32 tells scores apart by whole units only, each score rounded as the
  // reference it was taken for, and then their difference: as one operation the largest's own would be as far off 0.
  auto weights_of = [&](auto far, const f32x16& x, float off, Weights& w) __attribute__((always_inline)) {
    const bool apart = far && fabsf(off) >= 0x1p20f;  // (by row: the others keep their bits)
    float lx = 0.0f;
#pragma unroll
    for (int sb = 0; sb < 2; ++sb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = 8 * sb + 2 * e;
        auto less = [&](float y) { return CAP ? y - off : apart ? __builtin_fmaf(y, unit, 0.0f) - off : __builtin_fmaf(y, unit, -off); };
        put_weights<DT>(w, sb, e, fast_exp2(less(x[at])), fast_exp2(less(x[at + 1])), sb ? lx : l_run);
      }
    l_run += lx;
  };
  auto exponentials = [&](const f32x16& x, Weights& w) __attribute__((always_inline)) {
    const float off = m_ref == -INFINITY ? 0.0f : m_ref;
    if (!CAP && __builtin_expect(__any(fabsf(off) >= 0x1p20f), 0)) weights_of(std::true_type{}, x, off, w);
    else weights_of(std::false_type{}, x, off, w);
  };
  // A new reference where a score exceeds the old one by more than kSlack. What was weighed by the old one joins the accumulators
  // first; then they go over to the new one.
  auto move_reference = [&](float to, bool up) __attribute__((always_inline)) {
    const float c = m_ref == -INFINITY ? -1.0f : up ? fast_exp2(m_ref - to) : 1.0f;
    m_ref = up ? to : m_ref;
    l_run *= c;
    return c;
  };
  auto follow_reference = [&](float c) __attribute__((always_inline)) {
    // (Below 0 where there was none: whatever the accumulators hold goes.)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mfma_settle(acc[nt]);
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[nt][e] = c < 0.0f ? 0.0f : acc[nt][e] * c;
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
    const int ln = here(lane), key0 = key_of(h) + 16 * (wave & 1) + 8 * (ln >> 5);
    char* const mine_at = lds + (uint32_t(h) & (kRing - 1)) * L::kStage + wave * L::kRun + ln * 16;
    // (An exponent of ones, and only that, carries into the sign's place.)
    constexpr uint32_t kExp = DT == ESP_F16 ? 0x7c007c00u : 0x7f807f80u, kOne = DT == ESP_F16 ? 0x04000400u : 0x00800080u;
    uint32_t found = 0;
    const bool cut = key_of(h) < rg.from || key_of(h) + 32 > rg.end;
    uint32_t in[4] = {~0u, ~0u, ~0u, ~0u};
    if (cut) {
#pragma unroll
      for (int e = 0; e < 4; ++e) in[e] = in_range(key0 + 2 * e);
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const u32x4 v = *reinterpret_cast<const u32x4*>(mine_at + i * 1024);
#pragma unroll
      for (int e = 0; e < 4; ++e) found |= (v[e] & in[e] & kExp) + kOne;
    }
    const bool any = __any((found & 0x80008000u) != 0);
    if (cut || any) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        u32x4 v = *reinterpret_cast<const u32x4*>(mine_at + i * 1024);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] &= in[e];
          if (any) v[e] &= ~not_finite2<DT>(v[e]);
        }
        *reinterpret_cast<u32x4*>(mine_at + i * 1024) = v;
      }
    }
    if (ln == 0) bad[2 * (uint32_t(h) & (kRing - 1)) + (wave & 1)] = any;
  };
  bool marked;
  // A product of marks in such values' places with the keys that the rows see, which weigh something however little, says which outputs they reach.
  // (2048 rows behind 8000 keys, 32 / 8 heads: 520 us, 1330 with one infinite value, which is the second walk, 5300 with some in every stage.)
  auto marks = [&](int h) __attribute__((always_inline)) {
    const int ln = here(lane), lo = max(rg.from, sight.from), n = max(0, min(rg.end, sight.end) - lo);
    constexpr uint32_t one = DT == ESP_F16 ? 0x3c00u : 0x3f80u;
#pragma unroll 1
    for (int w = 0; w < NT; ++w) {
      uint32_t* const word = reinterpret_cast<uint32_t*>(lds + L::kMarks) + (wave * NT + w) * 64 + ln;
      uint32_t found = marked ? *word : 0u;
#pragma unroll 1
      for (int neg = 0; neg < 2; ++neg) {
        f32x16 seen = f32x16{};
#pragma unroll 1
        for (int key = key_of(h); key <= min(key_of(h) + 16, last_sub); key += 16) {
          const uint16_t* v = a.pool + size_t(a.kv_base) + (size_t(shaped_block(a, table, key / a.bt)) * size_t(a.Hkv) + size_t(kvh)) * head +
                              vt_elem(a.bt, HD, key % a.bt, 32 * w + (ln & 31)) + 8 * (ln >> 5);
          u32x4 x = *reinterpret_cast<const u32x4*>(v);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = not_finite_marks<DT>(x[e], neg != 0);
          u32x4 sees;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = key + 8 * (ln >> 5) + 2 * e - lo;
            sees[e] = (uint32_t(at) < uint32_t(n) ? one : 0u) | (uint32_t(at + 1) < uint32_t(n) ? one << 16 : 0u);
          }
          seen = mfma32x16<DT>(x, sees, seen);
          mfma_settle(seen);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) found |= seen[e] > 0.0f ? (neg ? 0x10000u : 1u) << e : 0u;
      }
      *word = found;
    }
    marked = true;
  };

  const int lead = kind == 0 ? 2 : 0;
  auto within = [](int h, int lo, int hi) { return uint32_t(h - lo) < uint32_t(hi - lo); };  // (lo <= hi)
  const float low_below = CAP ? a.tanh_below : 0.0f, short_below = CAP ? a.tanh_short : 0.0f;
  // Two turns between barriers: 64 keys. Behind the one in front of turns h and h + 1 (h even), K of stages h and h + 1 and V of stages h - 2
  // and h - 1 have landed for everybody, and nobody reads K or V of the two stages in front of those any more, whose places in the
  // ring the two turns' requests take.
  auto begin = [&](int h, bool edges) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (edges && kind == 1) {
#pragma unroll 1
      for (int x = max(h - 2, 0); x < min(h, n_st); ++x)
        if (!within(x, w0, w1)) mend(x);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // A turn of whatever there is to do, one after the other: S and W are the scores and the weights of the last stage.
  auto mixed_turn = [&](int h, f32x16& S, Weights& W) __attribute__((always_inline)) {
    // On a wavefront's first stage acc is whatever; it is cleared when a row's reference is first set.
    if (within(h - 2, v0, v1)) {
      weigh(h - 2, W, [](int) {});
      if (!within(h - 2, w0, w1)) {
        const int* f = bad + 2 * ((h - 2) & (kRing - 1));
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(f[0] | f[1]), 0)) marks(h - 2);
      }
    }
    if (within(h - 1, v0, v1)) {
      mfma_settle(S);
      const float b = bias_at(h - 1);
      // (Each score by its own size: those of keys that a row does not see may be anything, and choose nothing for the others.)
      const int lo = max(rg.from, sight.from), n = max(0, min(rg.end, sight.end) - lo);
      const int at0 = key_of(h - 1) + 8 * (here(lane) >> 5), at = at0 - lo;
      float mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int k = 16 * (e >> 3) + (e & 7);
        float x = CAP ? shaped_score<CAP>(a, S[e]) + bias[e] : S[e];
        if constexpr (BIAS) x += b - 2.0f * slope * fmaxf(float(at0 + k - qpos), 0.0f);
        S[e] = uint32_t(at + k) < uint32_t(n) ? x : -INFINITY;  // the row sees the keys [lo, lo + n)
        mx = fmaxf(mx, S[e]);
      }
      const float ref = reference_of<DT>(max_halves(mx) * unit);
      const bool up = ref - m_ref > kSlack;  // from -inf on: the first key that the row sees
      if (__any(up)) follow_reference(move_reference(ref, up));
      exponentials(S, W);
    }
    if (within(h, v0, v1)) {
      score(h, S, [](int) {});
      mfma_settle(S);
    }
  };
  // A turn with all three stages to do, the last two seen whole by all rows of the tile: scores of stage h to `to`, those of stage h - 1 in
  // `of`, weights of stage h - 2 in `had`, of stage h - 1 to `W`. No maximum is taken: all weights are positive, so a lane's sum bounds them, and only
  // where one is too large (or the row has no reference yet) does the reference move and the stage's weights are made again.
  auto whole_turn = [&](auto first, int h, f32x16& to, f32x16& of, const Weights& had, Weights& W) __attribute__((always_inline)) {
    const float stage = bias_at(h - 1) * unit;
    float off = m_ref - stage, sum[2] = {0.0f, 0.0f};
    auto weights = [&](int sb, bool apart) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = 8 * sb + 2 * e;
        auto less = [&](float x) { return apart ? __builtin_fmaf(x, unit, stage) - m_ref : CAP ? x - off : __builtin_fmaf(x, unit, -off); };
        put_weights<DT>(W, sb, e, fast_exp2(less(of[at])), fast_exp2(less(of[at + 1])), sum[sb]);
      }
    };
    auto made_here = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) asm volatile("" : "+v"(of[e]));
      if constexpr (!CAP) asm volatile("" : "+v"(W.p[0]), "+v"(W.rest[0]), "+v"(sum[0]));
    };
    // Under the score products: the scores' shape, or without a cap half of the weights.
    auto shaped = [&](auto terms) __attribute__((always_inline)) {
      score(h, to, [&](int g) __attribute__((always_inline)) {
        constexpr int PER = 16 / KS;
#pragma unroll
        for (int e = g * PER; e < (g + 1) * PER; ++e) of[e] = shape_e(of[e], e, terms);
        // Requests one by one: together at the turn's beginning they stand in line behind those of the other wavefronts.
        if (first && g % 2 == 1 && g < 2 * LOADS) request(h + lead, g / 2, 0);
      });
      if constexpr (!CAP) weights(0, false);
      lay_out<KS, 1, (CAP ? (terms == 3 ? 6 : 8) * 16 : 56) / KS>();
      made_here();
    };
    if constexpr (CAP) {
      const float largest = largest_size(of);
      if (__builtin_expect(!__any(!(largest < short_below)), 1)) shaped(std::integral_constant<int, 3>{});
      else if (!__any(!(largest < low_below))) shaped(std::integral_constant<int, 5>{});
      else shaped(std::integral_constant<int, 0>{});
    } else {
      shaped(std::integral_constant<int, 0>{});
    }
    look_up(first ? 0 : 1);
    weigh(h - 2, had, [&](int g) __attribute__((always_inline)) {
      if (first && g % 2 == 1 && g < 2 * LOADS) request(h + 1 + lead, g / 2, 1);
    });
    if constexpr (CAP) weights(0, false);
    weights(1, false);
    lay_out<2 * NT, 2, (CAP ? 104 : 56) / (4 * NT)>();
    asm volatile("" : "+v"(W.p[0]), "+v"(W.p[1]), "+v"(W.rest[0]), "+v"(W.rest[1]), "+v"(sum[0]), "+v"(sum[1]));  // (made here, not later)
    if (__builtin_expect(__any(!(sum[0] + sum[1] <= kMost<DT>)), 0)) {
      float mx = of[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, of[e]);
      mx = reference_of<DT>(max_halves(__builtin_fmaf(mx, unit, stage)));
      follow_reference(move_reference(mx, mx > m_ref));
      off = (m_ref == -INFINITY ? 0.0f : m_ref) - stage;
      const bool apart = fabsf(m_ref) >= 0x1p20f && m_ref != -INFINITY;
      sum[0] = sum[1] = 0.0f;
      weights(0, apart);
      weights(1, apart);
    }
    l_run += sum[0] + sum[1];
    if constexpr (!first) locate_both();
  };
  // Infinite and NaN values of a stage that all rows see whole go into its products as they are, and there an infinity makes NaN of a weight's
  // second number, or where a weight has vanished. Rows that have met such a value are walked once more, with all stages looked over as
  // those with unseen keys are; the tile's other rows are done.
  int* const met = bad + 2 * kRing;  // [wavefront]
  bool todo = col0 + l32 < cols_live;
  for (bool careful = false;; careful = true) {
    if (careful) f0 = f1 = w0 = w1 = 0;
    start();
    m_ref = -INFINITY;
    l_run = 0.0f;
    marked = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[nt] = f32x16{};
    // A pair of turns h and h + 1 requests stages h + lead and h + 1 + lead, both in the first turn, so that the barrier behind the second does
    // not wait for them (2048 rows behind 8000 keys, 16 / 8 heads of 256 dims, capped, with single weights: 393 to 378 us).
    {
      next_id[0] = block_id();
      at_t0[0] = next_t0;
      look_up(1);
      locate_both();
      if (kind == 0) {
        if (n_st > 0) request_all(0, 0);
        if (n_st > 1) request_all(1, 1);
        look_up(0);
        look_up(1);
        locate_both();
      }
    }
    // Q is waited for here, not at its first use in the loop: that wait would be on the counter of the stages on their way.
    // (Of 256 dims it lies in accumulation registers, which a product reads as well: in vector registers the longer forms of a cap spilled in
    // every stage, and waited for the stages on their way with it. 2048 rows behind 8000 keys, 16 / 8 heads, scores above 0.2 caps: 619 to 473 us.)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if constexpr (HD == 256) asm volatile("" : "+a"(qf[ks]));
      else asm volatile("" : "+v"(qf[ks]));
    }
    if (n_st > 0) {
      // Turns [t0, t1) are whole for this wavefront, in pairs.
      const int t0 = (max(max(f0 + 1, w0 + 2), v0 + 2) + 1) & ~1, t1 = max(t0, min(min(f1, w1) + 1, v1) & ~1);
      auto mixed_pair = [&](int h) __attribute__((always_inline)) {
        begin(h, true);
        if (h + lead < n_st) request_all(h + lead, 0);
        if (h + 1 + lead < n_st) request_all(h + 1 + lead, 1);
        look_up(0);
        look_up(1);
#pragma unroll 1
        for (int x = h; x < h + 2; ++x) mixed_turn(x, s[0], P[0]);
        locate_both();
      };
      int h = 0;
      for (; h < (t1 > t0 ? t0 : n_st + 2); h += 2) mixed_pair(h);
      for (; h < t1; h += 2) {
        begin(h, false);
        whole_turn(std::true_type{}, h, s[1], s[0], P[0], P[1]);
        whole_turn(std::false_type{}, h + 1, s[0], s[1], P[1], P[0]);
      }
      mfma_settle(s[0]);
      for (; h < n_st + 2; h += 2) mixed_pair(h);
    }

    // ---- the rows' end
    const int ln = here(lane), half = ln >> 5;
    const float l = l_run + __shfl_xor(l_run, 32);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mfma_settle(acc[nt]);
    bool again = false;
    if (!careful) {
      float nf[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 16; ++e) nf[e & 3] = __builtin_fmaf(acc[nt][e], 0.0f, nf[e & 3]);
      const float odd = (nf[0] + nf[1]) + (nf[2] + nf[3]);  // NaN, or 0
      again = todo && odd + __shfl_xor(odd, 32) != 0.0f;
      if (ln == 0) met[wave] = 0;
      if (again) met[wave] = 1;
    }
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
    __syncthreads();  // the ring is free
    const bool repeat = !careful && (met[0] | met[1] | met[2] | met[3]) != 0;
    const bool done = todo && !again;
    const bool none = l == 0.0f;  // a row that has seen nothing
    if (tile.part >= 0) {         // partial records
      if (done) {
        const size_t rec = (size_t(tile.part) * a.Hkv + kvh) * a.cols + col0 + (ln & 31);
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
      }
    } else {
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
      RowsOut<RB>::store(ob, done ? uint64_t(uintptr_t(a.O + size_t(tile.r0 + pl.m) * a.q_ld + size_t(kvh * a.G + pl.hg) * HD)) : 0, ln);
    }
    if (__builtin_expect(!repeat, 1)) return;
    todo = again;
    __syncthreads();  // the rows have left the ring
  }
}

namespace {

template <int DT, int HD, bool CAP, bool BIAS>
hipError_t launch_tiled_s(const ShapedArgs& a, int n_tiles, hipStream_t st) {
  constexpr auto k = attn_shaped_tiled_kernel<DT, HD, CAP, BIAS>;
  const hipError_t e = allow_dynamic_lds<k>(TiledLds<HD>::kBytes);
  if (e != hipSuccess || n_tiles == 0) return e;  // (no tiles: the limit alone)
  hipLaunchKernelGGL(k, dim3(unsigned(a.Hkv), unsigned(n_tiles)), dim3(256), size_t(TiledLds<HD>::kBytes), st, a);
  return hipGetLastError();
}

template <int DT, int HD>
hipError_t launch_tiled_t(const ShapedArgs& a, int n_tiles, hipStream_t st) {
  if (a.cap_log2 > 0.0f) return a.slopes ? launch_tiled_s<DT, HD, true, true>(a, n_tiles, st) : launch_tiled_s<DT, HD, true, false>(a, n_tiles, st);
  return a.slopes ? launch_tiled_s<DT, HD, false, true>(a, n_tiles, st) : launch_tiled_s<DT, HD, false, false>(a, n_tiles, st);
}

template <int DT, int HD>
hipError_t allow_tiled() {
  ShapedArgs a{};
  hipError_t e = launch_tiled_s<DT, HD, false, false>(a, 0, nullptr);
  if (e == hipSuccess) e = launch_tiled_s<DT, HD, false, true>(a, 0, nullptr);
  if (e == hipSuccess) e = launch_tiled_s<DT, HD, true, false>(a, 0, nullptr);
  if (e == hipSuccess) e = launch_tiled_s<DT, HD, true, true>(a, 0, nullptr);
  return e;
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
