// NF4 dequantization launch helper (kernel in nf4.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace esep {

struct Nf4Args {
  const void* packed;      // uint8 [n_blocks * 32]
  const uint8_t* absmax;   // uint8 [n_blocks]
  const float* absmax2;    // fp32 [ceil(n_blocks / 256)]
  const float* code2;      // fp32 [256]
  const float* offset;     // fp32 scalar (device)
  const float* nf4;        // fp32 [16]
  void* out;               // [n_blocks * 64] of the output dtype
  int64_t n_blocks;
};

constexpr int kNf4MultiMax = 8;

// Up to kNf4MultiMax weights decoded by one launch; weight i covers the global 4-packed-byte
// units [u0[i], u0[i + 1]) (8 per 64-element scale block).
struct Nf4Multi {
  Nf4Args w[kNf4MultiMax];
  int64_t u0[kNf4MultiMax + 1];
  int n;
};

hipError_t launch_nf4_dequant(const Nf4Multi& m, int out_dt, hipStream_t s, bool* supported);

// Products of up to kNf4MvRows rows x [M, K] with NF4 weights [N, K] that follow each other in the columns
// of y (nf4_matvec.hip).
constexpr int kNf4MvRows = 16;
struct Nf4MvWeight {
  const void* packed;
  const uint8_t* absmax;
  const float* absmax2;
  const float* code2;
  const float* offset;
  const float* nf4;
  const void* bias;  // [N] of x's type, or null
  int N;
  int col0;    // its first column of y
  int block0;  // its first block (the launcher's)
};
struct Nf4MvArgs {
  Nf4MvWeight w[kNf4MultiMax];
  int n;
  int per_block;  // tiles of 16 rows (the launcher's)
  const void* x;
  void* y;
  int64_t ldx, ldy;
  int M, K;
};

hipError_t launch_nf4_matvec(const Nf4MvArgs& a, int dt, hipStream_t s, bool* supported);

}  // namespace esep
