// Linear attention: what its kernels read, and the facts of their launches that the host planner counts with too. No device code.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../../include/espetero_attn.h"
#include "launch_shape.hpp"

namespace esp {

constexpr int kLinearChunk = 64;  // rows that the chunked kernel takes at a time
// Sequences of up to so many rows go through the recurrent kernel, whose time grows with every row beyond the state's own bytes. 32 heads of
// 128 x 128, bf16, recurrent and chunked: 64 sequences of 4 rows 46 and 56 us, of 8 56 and 56, of 12 66 and 55; one of 4 rows 5.6 and 9.3, of 8
// 6.3 and 9.1, of 12 8.0 and 9.2.
constexpr int kLinearFew = 8;

// Columns of V that a workgroup of the chunked kernel takes: P is made once more for every other 64. 128 and 64 columns, bf16, us, passes without
// a pause between them: four prompts of 2048 rows, 40 heads of 128 x 128, 157 and 194; 24 of 300, 32 heads, 91 and 120; one of 2000, 32 heads,
// 44 and 49, 8 heads 30 and 29.5.
constexpr int linear_cols(int dv) { return dv % 128 == 0 ? 128 : 64; }
constexpr bool linear_dims(int dk, int dv) { return (dk == 64 || dk == 128) && dv >= 64 && dv <= 512 && dv % 64 == 0; }

// Resident workgroups per compute unit of the chunked kernel: two of 78 KB of LDS, wavefronts of 256 registers (dk 64: by registers); of 64 x 64
// dims a third one fits, and fills what two leave.
constexpr int linear_workgroups_per_cu(int dk, int dv) { return dk == 64 && linear_cols(dv) == 64 ? 3 : 2; }

// Records of sequences cut into segments: states, then the log2 of what each segment's decays come to.
struct LinearCarve {
  size_t states, totals, total;
};
constexpr LinearCarve carve_linear(int H, int dk, int dv, int64_t n_parts) {
  const size_t recs = size_t(n_parts > 0 ? n_parts : 0) * size_t(H);
  LinearCarve c{};
  c.states = 0;
  c.totals = recs * size_t(dk) * size_t(dv) * sizeof(float);
  c.total = c.totals + recs * sizeof(double);
  return c;
}

// Everything a linear attention kernel reads, passed by value.
struct LinearArgs {
  const uint16_t* Q;
  const uint16_t* K;
  const uint16_t* V;
  const float* decay;
  float* states;
  uint16_t* O;
  const esp_linear_tile* tiles;
  float* parts;         // [part][H][dk dv], as the chunked kernel's lanes hold them
  double* part_totals;  // [part][H]
  int32_t H, group, dk, dv, q_ld, k_ld, v_ld, o_ld, decay_ld;  // group: heads that share a head of Q and K
  float scale;
};

}  // namespace esp
