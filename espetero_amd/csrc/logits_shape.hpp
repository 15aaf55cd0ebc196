// Argument block of the logits kernels and how a vocabulary becomes workgroups.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/espetero_attn.h"

namespace esp {

constexpr int kLogitsChunk = 8192;  // tokens of a workgroup where several share a row
constexpr int kLogitsSolo = 1024;   // threads of a workgroup that has a row to itself

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
// Whether a workgroup has a row to itself. A row's token joins a history that other rows may name too only when all rows have been
// read: with several rows that is the second launch's work.
constexpr bool logits_solo(int vocab, int n_rows, bool record) { return vocab <= 65536 && (n_rows == 1 || !record); }
constexpr size_t logits_workspace(int vocab, int n_rows) { return size_t(logits_chunks(vocab)) * size_t(n_rows) * 8; }

}  // namespace esp
