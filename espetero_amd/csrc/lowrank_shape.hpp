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
constexpr int kLowRankSplits = 8;  // at most
// How many ways D is split, with 128 dims or more each. Eight: a share for each XCD's L2, and what the second launch has on its way at
// once of a few rows. Four where that leaves enough workgroups, since every block of columns sums the splits again (3679 rows, rank 64,
// D 5120: 62 us, 67 with eight; 500 rows, rank 16, D 4096: 17 us, 15 with eight).
inline int lowrank_splits(int D, int n_low, int rows_per_tile, int n_tiles) {
  const int wgs = std::max(1, n_tiles * lowrank_low_groups(n_low));
  return std::max(1, std::min(D / 128, rows_per_tile == 16 ? std::min(kLowRankSplits, (512 + wgs - 1) / wgs) : wgs < 128 ? kLowRankSplits : 4));
}
// Whether one launch does both products, each workgroup the first one for itself: one launch less, and the slice's A read by every
// block of 1024 columns at what one compute unit draws. bf16, one request, D 2048, rank 16: 6.5 us; D 4096, rank 16: 8.9 us, 8.0 as two
// launches; 48 requests of 20 adapters, D 5120, rank 16: 12.7 us, 10.9 as two.
inline bool lowrank_fused(int D, int rank, int n_slices, const int32_t* width, int n_tiles) {
  int64_t wgs = 0;
  for (int s = 0; s < n_slices; ++s) wgs += (width[s] + 1023) / 1024;
  wgs *= n_tiles;
  return rank <= 32 && (wgs + 255) / 256 * rank * D <= 32 * 1024;
}
// Blocks of 128 columns that a workgroup of the second launch takes one after the other, with one sum of its tile's splits, as long as
// that leaves one and a quarter workgroups for every compute unit (2065 rows, rank 128, D 5120, 7168 columns: 58 us; 68 with one and a
// half, 66 with one or three. D 4096, 6144 columns: 50, 50, 58, 54).
constexpr int lowrank_blocks_each(int row_blocks, int n_tiles, int blocks) {
  return row_blocks == 1 ? 1 : std::max(1, std::min(8, int(int64_t(n_tiles) * blocks / 320)));
}
// Rows of a tile: a decode batch has few of each adapter.
constexpr int lowrank_rows(int n_rows) { return n_rows <= 0 ? 0 : n_rows <= 128 ? 16 : 64; }
// The intermediate of every split, as if there were always the most of them: what serves a pass serves every one of as many slots or
// fewer, whatever its tiles.
inline size_t lowrank_workspace(const esp_lowrank_params& p, int n_slots) {
  return size_t(std::max(1, std::min(p.D / 128, kLowRankSplits))) * size_t(n_slots) * size_t(p.n_slices * p.rank) * sizeof(float);
}
inline int lowrank_chunk(int D, int splits) { return ((D + splits - 1) / splits + 127) / 128 * 128; }

}  // namespace esp
