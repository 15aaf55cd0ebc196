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

// 16-row blocks of A that a workgroup of the first launch takes: all of them, or as even a share as there is of up to 4.
constexpr int lowrank_low_blocks(int n_low) {
  const int all = (n_low + 15) / 16, groups = (all + 3) / 4;
  return (all + groups - 1) / groups;
}
constexpr int lowrank_low_groups(int n_low) { return ((n_low + 15) / 16 + lowrank_low_blocks(n_low) - 1) / lowrank_low_blocks(n_low); }
// How many ways D is split, with 128 dims or more each: of few rows so often that the first launch has two workgroups for every
// compute unit, of many eight times, once for each XCD.
inline int lowrank_splits(int D, int n_low, int rows_per_tile, int n_tiles) {
  const int wgs = std::max(1, n_tiles * lowrank_low_groups(n_low)), want = rows_per_tile == 16 ? std::min(8, (512 + wgs - 1) / wgs) : 8;
  return std::max(1, std::min(D / 128, want));
}
// Whether one launch does both products, each workgroup of it the first one for itself.
inline bool lowrank_fused(int D, int rank, int n_slices, const int32_t* width, int n_tiles) {
  int64_t wgs = 0;
  for (int s = 0; s < n_slices; ++s) wgs += (width[s] + 1023) / 1024;
  wgs *= n_tiles;
  return rank <= 32 && (wgs + 255) / 256 * rank * D <= 32 * 1024;
}
// Blocks of columns that a workgroup of the second launch takes one after the other, with one sum of its tile's splits.
constexpr int lowrank_blocks_each(int row_blocks, int n_tiles, int blocks) {
  return row_blocks == 1 ? 1 : std::max(1, std::min(8, int(int64_t(n_tiles) * blocks / 512)));
}
constexpr int lowrank_rows(int n_rows) { return n_rows <= 0 ? 0 : n_rows <= 128 ? 16 : 64; }
inline size_t lowrank_workspace(const esp_lowrank_params& p, int n_tiles, int n_slots) {
  return size_t(lowrank_splits(p.D, p.n_slices * p.rank, p.rows_per_tile, n_tiles)) * size_t(n_slots) * size_t(p.n_slices * p.rank) * sizeof(float);
}
inline int lowrank_chunk(int D, int splits) { return ((D + splits - 1) / splits + 127) / 128 * 128; }

}  // namespace esp
