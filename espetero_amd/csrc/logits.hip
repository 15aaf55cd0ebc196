// The end of a decode step on the logits of its rows: the penalties for tokens that a request has seen, its biases, its grammar's
// mask, the best token that is left, and that token's entry in the request's history.
//
// Bound by HBM: a logit is read once and, where the caller wants them back, written once; the histories' two bits a token come
// with them. The counts behind the bits are read only where a bit is set, and then cost a line each: 192 fp32 rows of 250000 tokens with
// up to 6000 seen move 309 MB in 47 us, 6.6 TB/s, 74 MB of it for counts (50 to 58 us with the second launch, 107 where the logits are
// wanted back, another 192 MB). Small passes are bound by the hops to a row's record, its words and its counts, and by the second launch:
// 48 bf16 rows of 50257 take 11 to 13 us (8 + 3 in the kernels), one fp32 row of 32000 takes 7 to 8.5.
#include "common.hpp"
#include "logits_shape.hpp"

namespace esp {

namespace {

struct Best {
  float v;
  int32_t t;
};
// The larger logit; of equal ones the lower token.
__device__ __forceinline__ Best better(Best a, Best b) { return (b.v > a.v || (b.v == a.v && b.t < a.t)) ? b : a; }

__device__ __forceinline__ Best wave_best(Best b) {
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) b = better(b, Best{__shfl_xor(b.v, x), __shfl_xor(b.t, x)});
  return b;
}

template <int DT>
__device__ __forceinline__ float logit_at(const void* L, size_t i) {
  if constexpr (DT == ESP_F32) return static_cast<const float*>(L)[i];
  else return unpack_lo<DT>(static_cast<const uint16_t*>(L)[i]);
}
// 16 bytes at any address, and the logit e of them.
__device__ __forceinline__ u32x4 load16(const char* p) {
  u32x4 v;
  __builtin_memcpy(&v, p, 16);
  return v;
}
template <int DT>
__device__ __forceinline__ float logit_of(u32x4 v, int e) {
  if constexpr (DT == ESP_F32) return __uint_as_float(v[e]);
  else return e & 1 ? unpack_hi<DT>(v[e >> 1]) : unpack_lo<DT>(v[e >> 1]);
}

}  // namespace

// One logit through the penalties: the operations in this order and each rounded by itself, so that equal inputs give equal logits
// wherever they are computed.
__device__ __forceinline__ float penalised(float x, bool known, bool given, int count, float repetition, float frequency, float presence) {
#pragma clang fp contract(off)
  if (known) x = x > 0.0f ? x / repetition : x * repetition;
  if (given) {
    const float n = frequency * float(count);
    x = x - n;
    x = x - presence;
  }
  return x;
}

__device__ __forceinline__ void record_token(uint32_t* seen, int32_t* counts, int vocab, int words, int n_slots, int slot, int t, bool given) {
  if (slot < 0 || slot >= n_slots || t < 0 || t >= vocab) return;
  atomicOr(seen + (size_t(slot) * 2 + (given ? 1 : 0)) * words + t / 32, 1u << (t & 31));
  if (given) atomicAdd(counts + size_t(slot) * vocab + t, 1);
}

// grid: (chunks of 256 TP tokens, rows). The penalties touch few of the tokens, and so do the biases: their bits are gathered first,
// and a chunk's tokens then go two ways. The many that nothing but the mask touches are passed on and compared as they come. The few
// others become a list in LDS that all lanes share, whichever thread's they were, since a lane that found one among its own would hold
// up 63 that found none: done in place, with the counts behind it, 192 rows of 250000 took 126 us where they now take 50 to 58.
template <int DT, bool OUT, int TP>
__global__ __launch_bounds__(256) void logits_kernel(const LogitsArgs a) {
  constexpr int W = 256, CH = TP * W, NW = CH / 32;                  // threads, tokens of a chunk, its words of bits
  constexpr int VT = DT == ESP_F32 ? 4 : 8, U = TP / VT, B = 4;      // tokens of a load, loads of a thread, listed tokens of it at once
  static_assert(U >= 1 && NW <= W);
  __shared__ uint16_t list[CH];
  __shared__ uint32_t skip_sh[NW + 1], allowed_sh[NW + 1], known_sh[NW], given_sh[NW], biased_sh[NW];
  __shared__ float best_sh[W / 64];
  __shared__ int n_list, token_sh;
  const int row = blockIdx.y, tid = threadIdx.x, c0 = blockIdx.x * CH, n = min(CH, a.vocab - c0);  // the chunk has n tokens
  const char* const in = static_cast<const char*>(a.logits) + (size_t(row) * a.in_ld + c0) * (16 / VT);
  float* const out = OUT ? a.out + size_t(row) * a.out_ld + c0 : nullptr;
  // The logits are on their way before the row's record is here. A load that would reach over the chunk's end is moved back to end
  // there, and those behind it do the same again: nothing comes of seeing a token twice, and no load waits for a branch.
  auto at = [&](int u) { return max(0, min((u * W + tid) * VT, n - VT)); };
  auto few = [&] {  // a vocabulary, or the last of it, of fewer tokens than a load has
    u32x4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == ESP_F32) {
        v[e] = e < n ? reinterpret_cast<const uint32_t*>(in)[e] : 0u;
      } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(in) + 2 * e;
        v[e] = (2 * e < n ? p[0] : 0u) | (2 * e + 1 < n ? uint32_t(p[1]) << 16 : 0u);
      }
    }
    return v;
  };
  u32x4 x[U];
  if (n >= VT) {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = load16(in + uint32_t(at(u) * (16 / VT)));
  } else {
    x[0] = few();
#pragma unroll
    for (int u = 1; u < U; ++u) x[u] = x[0];
  }
  __builtin_amdgcn_sched_barrier(0);
  const esp_logits_row r = a.rows[row];
  const bool hist = r.slot >= 0 && r.slot < a.n_slots, masked = r.mask >= 0 && r.mask < a.n_masks;
  const uint32_t* const prompt = a.seen + (hist ? size_t(r.slot) * 2 * a.words : 0);
  const int32_t* const counts = a.counts + (hist ? size_t(r.slot) * a.vocab : 0) + c0;
  const uint32_t* const mask = a.masks + (masked ? size_t(r.mask) * a.words : 0);
  // The row's bias entries that there are.
  const int64_t e0 = max(r.bias0, 0), e1 = min(int64_t(a.n_bias), int64_t(r.bias0) + r.n_bias);
  const int n_bias = r.n_bias > 0 && e1 > e0 ? int(e1 - e0) : 0;
  const int32_t* const bias_tokens = a.bias_tokens + (n_bias ? e0 : 0);
  const float* const bias_values = a.bias_values + (n_bias ? e0 : 0);
  // Thread i's word of 32 tokens, and its first bias entry.
  const int w = min(c0 / 32 + tid, a.words - 1), left = tid < NW ? n - 32 * tid : 0;
  const uint32_t real = left >= 32 ? ~0u : left > 0 ? (1u << left) - 1 : 0u;
  uint32_t known = 0, given = 0, allowed = ~0u, first = ~0u;
  float plus = 0.0f;
  if (hist) known = prompt[w], given = prompt[a.words + w];
  if (masked) allowed = mask[w];
  if (n_bias) {
    const int e = min(tid, n_bias - 1);
    first = uint32_t(bias_tokens[e]) - uint32_t(c0);
    plus = bias_values[e];
  }
  if (tid < NW) biased_sh[tid] = 0;
  if (tid == 0) n_list = 0, token_sh = INT32_MAX, skip_sh[NW] = allowed_sh[NW] = 0;
  given &= real;
  known = (known & real) | given;
  allowed &= real;
  if (tid >= n_bias) first = ~0u;
  __syncthreads();
  if (n_bias) {  // the same for the whole workgroup
    for (int e = tid; e < n_bias; e += W) {
      const uint32_t t = e == tid ? first : uint32_t(bias_tokens[e]) - uint32_t(c0);
      if (t < uint32_t(n)) atomicOr(&biased_sh[t >> 5], 1u << (t & 31));
    }
    __syncthreads();
  }
  if (tid < NW) {
    const uint32_t biased = biased_sh[tid];
    uint32_t mine = known & allowed & ~biased;
    allowed_sh[tid] = allowed;
    known_sh[tid] = known;
    given_sh[tid] = given;
    skip_sh[tid] = known | biased | ~allowed;
    // Where in the list the thread's tokens go: behind those of the lanes below, and those behind the other wavefronts' as they come.
    const int lane = tid & 63, have = __popc(mine), lanes = min(NW, 64);
    int upto = have;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int below = __shfl_up(upto, d);
      if (lane >= d) upto += below;
    }
    int to = 0;
    if (lane == lanes - 1) to = atomicAdd(&n_list, upto);
    for (to = __shfl(to, lanes - 1) + upto - have; mine; mine &= mine - 1) list[to++] = uint16_t(32 * tid + __ffs(mine) - 1);
  }
  __syncthreads();
  auto bits_at = [&](const uint32_t* sh, int i) { return uint32_t((uint64_t(sh[(i >> 5) + 1]) << 32 | sh[i >> 5]) >> (i & 31)); };
  // The tokens that nothing but the mask touches.
  float most = -INFINITY;
  int where = 0;  // the largest of them, and where its load began
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t skip = bits_at(skip_sh, at(u));
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < VT; ++e) top = fmaxf(top, skip >> e & 1 ? -INFINITY : logit_of<DT>(x[u], e));
    where = top > most ? at(u) : where;
    most = fmaxf(most, top);
    if constexpr (OUT) {
      const uint32_t ok = bits_at(allowed_sh, at(u));
      float y[VT];
#pragma unroll
      for (int e = 0; e < VT; ++e) y[e] = ok >> e & 1 ? logit_of<DT>(x[u], e) : -INFINITY;
      if (n >= VT) {
        if ((u * W + tid) * VT < n) __builtin_memcpy(out + uint32_t(at(u)), y, sizeof y);
      } else {
#pragma unroll
        for (int e = 0; e < VT; ++e)
          if (e < n) out[e] = y[e];
      }
    }
  }
  if constexpr (OUT) __syncthreads();  // what follows writes over some of these
  // The others; past the list's end the last again, read but not written: in place it may have its penalty by then.
  Best other{-INFINITY, INT32_MAX};
  auto bit_of = [&](const uint32_t* sh, int i) { return (sh[i >> 5] >> (i & 31) & 1) != 0; };
  auto given_times = [&](int i) { return counts[bit_of(given_sh, i) ? uint32_t(i) : 0u]; };
  auto penalty = [&](float v, int i, bool known, int times) {
    return penalised(v, known, bit_of(given_sh, i), times, r.repetition, r.frequency, r.presence);
  };
  auto done = [&](int i, float y) {
    if constexpr (OUT) out[uint32_t(i)] = y;
    other = better(other, Best{y, c0 + i});
  };
  const int listed = n_list;
  for (int k = tid; k < listed; k += B * W) {
    int i[B], times[B];
    float v[B];
#pragma unroll
    for (int j = 0; j < B; ++j) i[j] = list[min(k + j * W, listed - 1)];
#pragma unroll
    for (int j = 0; j < B; ++j) v[j] = logit_at<DT>(in, uint32_t(i[j])), times[j] = given_times(i[j]);
#pragma unroll
    for (int j = 0; j < B; ++j)
      if (k + j * W < listed) done(i[j], penalty(v[j], i[j], true, times[j]));
  }
  for (int e = tid; e < n_bias; e += W) {
    const uint32_t t = e == tid ? first : uint32_t(bias_tokens[e]) - uint32_t(c0);
    if (t >= uint32_t(n) || !bit_of(allowed_sh, int(t))) continue;
    const float v = penalty(logit_at<DT>(in, t), int(t), bit_of(known_sh, int(t)), hist ? given_times(int(t)) : 0);
    done(int(t), v + (e == tid ? plus : bias_values[e]));
  }
  if (!a.tokens) return;  // the same for every workgroup
  float v = fmaxf(most, other.v);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  if ((tid & 63) == 0) best_sh[tid >> 6] = v;
  __syncthreads();
  v = fmaxf(fmaxf(best_sh[0], best_sh[1]), fmaxf(best_sh[2], best_sh[3]));
  // Only lanes that hold the chunk's best logit look for its token, in the load that it came with.
  if (v > -INFINITY) {
    int t = other.v == v ? other.t : INT32_MAX;
    if (most == v) {
      const u32x4 again = n >= VT ? load16(in + uint32_t(where * (16 / VT))) : few();
      const uint32_t skip = bits_at(skip_sh, where);
#pragma unroll
      for (int e = VT - 1; e >= 0; --e) t = (int(~skip >> e & 1) & int(logit_of<DT>(again, e) == v)) ? min(t, c0 + where + e) : t;
    }
    if (t != INT32_MAX) atomicMin(&token_sh, t);
  }
  __syncthreads();
  if (tid != 0) return;
  a.part_v[size_t(row) * gridDim.x + blockIdx.x] = v;
  a.part_t[size_t(row) * gridDim.x + blockIdx.x] = token_sh;
}

// One wavefront per row: the best of the chunks' best.
__global__ __launch_bounds__(64) void logits_pick_kernel(const LogitsArgs a, int chunks) {
  const int row = blockIdx.x, slot = a.record ? a.rows[row].slot : -1;
  Best best{-INFINITY, INT32_MAX};
  for (int c = threadIdx.x; c < chunks; c += 64) best = better(best, Best{a.part_v[size_t(row) * chunks + c], a.part_t[size_t(row) * chunks + c]});
  best = wave_best(best);
  if (threadIdx.x != 0) return;
  const int t = best.v > -INFINITY ? best.t : -1;
  a.tokens[row] = t;
  record_token(a.seen, a.counts, a.vocab, a.words, a.n_slots, slot, t, true);
}

__global__ __launch_bounds__(256) void history_record_kernel(uint32_t* seen, int32_t* counts, const int32_t* tokens, const int32_t* slots, int n,
                                                             int vocab, int words, int n_slots, int given) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) record_token(seen, counts, vocab, words, n_slots, slots[i], tokens[i], given != 0);
}

__global__ __launch_bounds__(256) void history_clear_kernel(uint32_t* seen, int32_t* counts, const int32_t* slots, int vocab, int words, int n_slots) {
  const int slot = slots[blockIdx.y];
  if (slot < 0 || slot >= n_slots) return;
  for (int i = blockIdx.x * 256 + threadIdx.x; i < max(vocab, 2 * words); i += gridDim.x * 256) {
    if (i < vocab) counts[size_t(slot) * vocab + i] = 0;
    if (i < 2 * words) seen[size_t(slot) * 2 * words + i] = 0;
  }
}

template <int DT, int TP>
static void run_logits(const LogitsArgs& a, const LogitsShape& s, int n_rows, hipStream_t st) {
  const dim3 grid{unsigned(s.chunks), unsigned(n_rows)}, block{256};
  if (a.out) hipLaunchKernelGGL((logits_kernel<DT, true, TP>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((logits_kernel<DT, false, TP>), grid, block, 0, st, a);
}

template <int DT>
static void run_logits(const LogitsArgs& a, const LogitsShape& s, int n_rows, hipStream_t st) {
  if (s.tokens == 8) run_logits<DT, 8>(a, s, n_rows, st);
  else run_logits<DT, 16>(a, s, n_rows, st);
}

hipError_t launch_logits(int dt, const LogitsArgs& a, int n_rows, hipStream_t st) {
  const LogitsShape s = logits_shape(a.vocab, n_rows);
  if (dt == ESP_F32) run_logits<ESP_F32>(a, s, n_rows, st);
  else if (dt == ESP_F16) run_logits<ESP_F16>(a, s, n_rows, st);
  else run_logits<ESP_BF16>(a, s, n_rows, st);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.tokens) return e;
  hipLaunchKernelGGL(logits_pick_kernel, dim3(unsigned(n_rows)), dim3(64), 0, st, a, s.chunks);
  return hipGetLastError();
}

hipError_t launch_history_record(const esp_logits_params* p, uint32_t* seen, int32_t* counts, const int32_t* tokens, const int32_t* slots, int n,
                                 int given, hipStream_t st) {
  hipLaunchKernelGGL(history_record_kernel, dim3(unsigned((n + 255) / 256)), dim3(256), 0, st, seen, counts, tokens, slots, n, p->vocab,
                     logits_words(p->vocab), p->n_slots, given);
  return hipGetLastError();
}

hipError_t launch_history_clear(const esp_logits_params* p, uint32_t* seen, int32_t* counts, const int32_t* slots, int n, hipStream_t st) {
  hipLaunchKernelGGL(history_clear_kernel, dim3(unsigned(std::min(64, (p->vocab + 255) / 256)), unsigned(n)), dim3(256), 0, st, seen, counts, slots,
                     p->vocab, logits_words(p->vocab), p->n_slots);
  return hipGetLastError();
}

}  // namespace esp
