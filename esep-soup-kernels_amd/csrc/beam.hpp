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
  int R, W, V, keep, splits;
  int piece, each;  // elements that a block has room for, and that it takes: pieces of one size, as few values bound nothing
};

// Candidates that a thread of the join (of 1024) asks for at once.
constexpr int kBeamJoinFirst = 4;
// Elements of a row that a block takes: few, so that short launches fill the card, until that would make more than
// 1024 blocks or more candidates than the join takes at once. Pieces of 2048 / 4096 / 8192, both launches in us: 1 x
// 4 x 151936 bf16, keep 8 9.2 / 9.0 / 9.5; 16 x 4 x 50001 12.4 / 12.9 / 13.5; 24 x 5 x 151936 fp32, keep 5 26.5 /
// 21.7 / 22.2; 8 x 8 x 151936 bf16, keep 16 24.2 / 17.1 / 15.4; 128 x 4, keep 8 77 / 53 / 47; 1 x 8 x 151936, keep 16
// 15.1 / - / 11.3, keep 64 70 / - / 22.
inline int beam_piece(int64_t R, int W, int64_t V, int keep) {
  int piece = kBeamThreads * 8;
  while (piece < kBeamThreads * 32) {
    const int64_t splits = (V + piece - 1) / piece;
    if (R * W * splits <= 1024 && W * splits * keep <= 1024 * kBeamJoinFirst) break;
    piece *= 2;
  }
  return piece;
}
inline int64_t beam_splits(int64_t R, int W, int64_t V, int keep) {
  const int p = beam_piece(R, W, V, keep);
  return (V + p - 1) / p;
}

hipError_t launch_beam_select(const BeamArgs& a, int dt, hipStream_t s, bool* supported);

}  // namespace esep
