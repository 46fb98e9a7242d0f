// Launch helpers of the paged caches' upkeep (kernels in paged.hip): block tables and slots, the store of new keys
// and values, the reordering of beams.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace esep {

struct PageTablesArgs {
  int32_t* tables;         // [B, M] by t_bs
  const int32_t* lengths;  // [B] tokens in each row before
  const int32_t* add;      // [B] tokens to add
  const int32_t* free;     // [F] pages to take, from free[*taken] on
  const int32_t* taken;    // [1]
  int32_t* slots;          // [total]
  int32_t* positions;      // [total]
  int32_t* cu;             // [B + 1]
  int32_t* lengths_out;    // [B], may be lengths
  int32_t* taken_out;      // [1], may be taken
  int64_t t_bs;
  int B, M, F, P, total;
};
hipError_t launch_page_tables(const PageTablesArgs& a, hipStream_t s);

// K and V caches in pages: token t of page i, head h at i * ps + t * ts + h * hs elements of 16 bits (layer l: + l * ls).
struct Pages {
  void* p;
  int64_t ls, ps, ts, hs;
};
struct PageStoreArgs {
  const void* src[2];  // [T, HK, D] by (s_ts, s_hs)
  int64_t s_ts[2], s_hs[2];
  Pages dst[2];
  const int32_t* slots;  // [T]
  int64_t T;
  int N, P, HK, D;
};
hipError_t launch_page_store(const PageStoreArgs& a, hipStream_t s);

constexpr int kMostBeams = 32;
struct BeamReorderArgs {
  const int32_t* parents;  // [R, W]
  const int32_t* tables;   // [R * W, M] by t_bs
  const int32_t* lengths;  // [R]
  const int32_t* start;    // [R] or null (0)
  Pages pages[2];
  int64_t t_bs;
  int R, W, M, N, P, L, HK, D;
};
hipError_t launch_beam_reorder(const BeamReorderArgs& a, hipStream_t s);

}  // namespace esep
