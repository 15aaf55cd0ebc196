// Argument block of the low-rank adapter kernels and how a pass becomes workgroups.
#pragma once

#include <algorithm>
#include <cstddef>
#include <cstdint>

#include "../../include/espetero_attn.h"

namespace esp {

constexpr int kLowRankMost = 128;  // largest rank

struct LowRankArgs {
  const uint16_t* X;
  const uint16_t* A;   // [adapter][slices * rank][D]
  const uint16_t* B;   // [adapter][columns of all slices][rank]
  const float* scale;  // [adapter]
  float* Y;
  const int32_t* order;
  const esp_lowrank_tile* tiles;
  float* low;          // [split][slot][slices * rank]
  int32_t D, rank, n_slices, n_low, n_out, x_ld, y_ld, n_slots, splits, chunk;
  int32_t y_off[ESP_LOWRANK_SLICES], width[ESP_LOWRANK_SLICES];
};

// How many ways D is split: so many that the first launch has two workgroups for every compute unit, each with 256 dims or more.
inline int lowrank_splits(int D, int n_tiles) {
  const int most = std::max(1, D / 256), want = std::max(1, 512 / std::max(1, n_tiles));
  return std::min(most, want);
}
constexpr int lowrank_rows(int n_rows) { return n_rows > 0 ? 16 : 0; }
inline size_t lowrank_workspace(const esp_lowrank_params& p, int n_tiles, int n_slots) {
  return size_t(lowrank_splits(p.D, n_tiles)) * size_t(n_slots) * size_t(p.n_slices * p.rank) * sizeof(float);
}
inline int lowrank_chunk(int D, int splits) { return ((D + splits - 1) / splits + 31) / 32 * 32; }

}  // namespace esp
