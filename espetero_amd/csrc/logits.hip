// The end of a decode step on the logits of its rows: the penalties for tokens that a request has seen, its biases, its grammar's
// mask, the best token that is left, and that token's entry in the request's history.
//
// Bound by HBM: a logit is read once and, where the caller wants them back, written once; the histories' two bits a token come
// with them. The counts behind the bits are read only where a bit is set. A thread takes 8 consecutive tokens, whose bits are one
// byte of each bit array.
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

template <int DT, bool OUT>
__global__ __launch_bounds__(256) void logits_kernel(const LogitsArgs a) {
  __shared__ float bias[kLogitsChunk];
  __shared__ Best best_sh[4];
  const int row = blockIdx.y, c0 = blockIdx.x * kLogitsChunk;
  const esp_logits_row r = a.rows[row];
  const bool hist = r.slot >= 0 && r.slot < a.n_slots;
  const uint8_t* prompt = hist ? reinterpret_cast<const uint8_t*>(a.seen + size_t(r.slot) * 2 * a.words) : nullptr;
  const uint8_t* given = hist ? prompt + size_t(a.words) * 4 : nullptr;
  const int32_t* counts = hist ? a.counts + size_t(r.slot) * a.vocab : nullptr;
  const uint8_t* mask = r.mask >= 0 && r.mask < a.n_masks ? reinterpret_cast<const uint8_t*>(a.masks + size_t(r.mask) * a.words) : nullptr;
  // The row's bias entries that fall into this chunk.
  const int e0 = max(r.bias0, 0), e1 = r.n_bias > 0 ? int(min(int64_t(a.n_bias), int64_t(r.bias0) + r.n_bias)) : e0;
  bool any = false;
  if (e1 > e0) {  // the same for the whole workgroup
    for (int i = threadIdx.x; i < kLogitsChunk; i += 256) bias[i] = 0.0f;
    __syncthreads();
    for (int e = e0 + int(threadIdx.x); e < e1; e += 256) {
      const int t = a.bias_tokens[e] - c0;
      if (t >= 0 && t < kLogitsChunk) {
        bias[t] = a.bias_values[e];
        any = true;
      }
    }
    any = __syncthreads_or(any);
  }
  Best best{-INFINITY, INT32_MAX};
  for (int i = threadIdx.x * 8; i < kLogitsChunk; i += 256 * 8) {
    const int t0 = c0 + i, n = min(8, a.vocab - t0);
    if (n <= 0) break;
    const uint32_t pb = hist ? prompt[t0 / 8] : 0u, gb = hist ? given[t0 / 8] : 0u, mb = mask ? mask[t0 / 8] : 255u;
    for (int e = 0; e < n; ++e) {
      const int t = t0 + e;
      float x = logit_at<DT>(a.logits, size_t(row) * a.in_ld + t);
      const bool gv = gb >> e & 1, kn = gv || (pb >> e & 1);
      x = penalised(x, kn, gv, gv ? counts[t] : 0, r.repetition, r.frequency, r.presence);
      if (any && e1 > e0) x = x + bias[i + e];
      if (!(mb >> e & 1)) x = -INFINITY;
      if constexpr (OUT) a.out[size_t(row) * a.out_ld + t] = x;
      if (x > best.v) best = Best{x, t};
    }
  }
  best = wave_best(best);
  if ((threadIdx.x & 63) == 0) best_sh[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    best = better(better(best_sh[0], best_sh[1]), better(best_sh[2], best_sh[3]));
    a.part_v[size_t(row) * gridDim.x + blockIdx.x] = best.v;
    a.part_t[size_t(row) * gridDim.x + blockIdx.x] = best.t;
  }
}

__device__ __forceinline__ void record_token(uint32_t* seen, int32_t* counts, int vocab, int words, int n_slots, int slot, int t, bool given) {
  if (slot < 0 || slot >= n_slots || t < 0 || t >= vocab) return;
  atomicOr(seen + (size_t(slot) * 2 + (given ? 1 : 0)) * words + t / 32, 1u << (t & 31));
  if (given) atomicAdd(counts + size_t(slot) * vocab + t, 1);
}

// One wavefront per row: the best of the chunks' best.
__global__ __launch_bounds__(64) void logits_pick_kernel(const LogitsArgs a, int chunks) {
  const int row = blockIdx.x;
  Best best{-INFINITY, INT32_MAX};
  for (int c = threadIdx.x; c < chunks; c += 64) best = better(best, Best{a.part_v[size_t(row) * chunks + c], a.part_t[size_t(row) * chunks + c]});
  best = wave_best(best);
  if (threadIdx.x != 0) return;
  const int t = best.t == INT32_MAX ? -1 : best.t;
  a.tokens[row] = t;
  if (a.record) record_token(a.seen, a.counts, a.vocab, a.words, a.n_slots, a.rows[row].slot, t, true);
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

hipError_t launch_logits(int dt, const LogitsArgs& a, int n_rows, hipStream_t st) {
  const int chunks = logits_chunks(a.vocab);
  const dim3 grid{unsigned(chunks), unsigned(n_rows)}, block{256};
  if (a.out) {
    if (dt == ESP_F32) hipLaunchKernelGGL((logits_kernel<ESP_F32, true>), grid, block, 0, st, a);
    else if (dt == ESP_F16) hipLaunchKernelGGL((logits_kernel<ESP_F16, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((logits_kernel<ESP_BF16, true>), grid, block, 0, st, a);
  } else {
    if (dt == ESP_F32) hipLaunchKernelGGL((logits_kernel<ESP_F32, false>), grid, block, 0, st, a);
    else if (dt == ESP_F16) hipLaunchKernelGGL((logits_kernel<ESP_F16, false>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((logits_kernel<ESP_BF16, false>), grid, block, 0, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.tokens) return e;
  hipLaunchKernelGGL(logits_pick_kernel, dim3(unsigned(n_rows)), dim3(64), 0, st, a, chunks);
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
