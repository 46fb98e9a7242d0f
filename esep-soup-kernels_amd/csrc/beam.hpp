// Launch helper of beam search's selection (kernels in beam.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace esep {

constexpr int kBeamMostKeep = 64;
constexpr int kBeamThreads = 256;

struct BeamArgs {
  const void* logits;   // [R, W, V] by (r_bs, w_bs)
  const float* scores;  // [R, W]
  float2* stat;         // [R W, splits] maximum and sum of the exponentials of a piece of a row
  uint64_t* cand;       // [R W, splits, keep] its candidates, the best first, 0 behind the last
  float* out_scores;    // [R, keep]
  int32_t* out_parents;
  int32_t* out_tokens;
  int64_t r_bs, w_bs;
  int R, W, V, keep, splits, piece;
};

// Elements of a row that a block takes.
inline int beam_piece(int64_t rows, int64_t V) {
  int piece = kBeamThreads * 8;
  while (piece < kBeamThreads * 32 && rows * ((V + piece - 1) / piece) > 1024) piece *= 2;
  return piece;
}
inline int64_t beam_splits(int64_t rows, int64_t V) {
  const int p = beam_piece(rows, V);
  return (V + p - 1) / p;
}

hipError_t launch_beam_select(const BeamArgs& a, int dt, bool vec, hipStream_t s, bool* supported);

}  // namespace esep
