// Argument block of the logits kernels and how a vocabulary becomes workgroups.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/espetero_attn.h"

namespace esp {

struct LogitsArgs {
  const void* logits;
  float* out;
  int32_t* tokens;
  const esp_logits_row* rows;
  const int32_t* bias_tokens;
  const float* bias_values;
  const uint32_t* masks;
  uint32_t* seen;    // [slot][prompt | given][words]
  int32_t* counts;   // [slot][vocab]
  float* part_v;     // [row][chunk]
  int32_t* part_t;
  int32_t vocab, words, in_ld, out_ld, n_slots, n_masks, n_bias, record;
};

constexpr int logits_words(int vocab) { return (vocab + 31) / 32; }
// Tokens of a thread and the chunks of 256 times as many that a row becomes: a small pass has as many workgroups as it can, a large one
// less to do for each beside its tokens.
struct LogitsShape {
  int tokens, chunks;
};
constexpr int kLogitsTokensLeast = 8;
constexpr int logits_chunks(int vocab, int tokens) { return (vocab + 256 * tokens - 1) / (256 * tokens); }
inline LogitsShape logits_shape(int vocab, int n_rows) {
  const int tokens = int64_t(vocab) * n_rows <= 12 << 20 ? kLogitsTokensLeast : 16;
  return {tokens, logits_chunks(vocab, tokens)};
}
// A best token of every chunk. As if the chunks were always the small ones: what serves a pass serves every smaller one.
inline size_t logits_workspace(int vocab, int n_rows) { return size_t(logits_chunks(vocab, kLogitsTokensLeast)) * size_t(n_rows) * 8; }

}  // namespace esp
