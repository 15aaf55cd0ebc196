// Argument block of the logits kernels and how a vocabulary becomes workgroups.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/espetero_attn.h"

namespace esp {

constexpr int kLogitsChunk = 2048;  // tokens of a workgroup

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
constexpr int logits_chunks(int vocab) { return (vocab + kLogitsChunk - 1) / kLogitsChunk; }
constexpr size_t logits_workspace(int vocab, int n_rows) { return size_t(logits_chunks(vocab)) * size_t(n_rows) * 8; }

}  // namespace esp
