// Attention of the newest tokens over a paged cache (attention_paged.hip): arguments and sizes.
#pragma once

#include "attention.hpp"

namespace esep {

struct AttnPagedArgs {
  const void* q;          // [B, n, HQ, D] by (q_bs, q_ts, q_hs)
  const void* k;          // [N, P, HK, D] by (k_ps, k_ts, k_hs)
  const void* v;
  void* o;                // [B, n, HQ, D] dense
  const int32_t* tables;  // [B, M] by t_bs: the pages of each row's tokens
  const int32_t* len;     // [B] tokens in each row's pages, the n new ones last
  const int32_t* shared;  // [B / W] first tokens that W rows in turn hold in the same pages, or null
  int2* ends;             // [groups] first and last wavefront of each group
  float* part;            // partials behind them
  int64_t q_bs, q_ts, q_hs, k_ps, k_ts, k_hs, v_ps, v_ts, v_hs, t_bs;
  int B, n, W, M, N, HQ, HK;
  int page_shift;         // P = 1 << page_shift, at least 16
  int window, sinks;      // window at least 1; none: M P
  float scale_log2;
  __host__ __device__ int tokens() const { return M << page_shift; }
};

// Groups are (rows that are walked together, kv head, 32 query rows of theirs): each row on its own, and before
// them, with shared pages, each W rows together over what they share.
struct PagedSizes {
  int64_t rows, row_tiles;      // query rows of a kv head on their own, tiles of 32 of them
  int64_t all_rows, all_tiles;  // of W rows together
  int64_t shared_groups, groups, tiles, units, floats;
};
inline PagedSizes paged_sizes(int B, int n, int W, int S, int HQ, int HK, int D, int window, int sinks,
                              bool shared) {
  PagedSizes z{};
  z.rows = (int64_t)n * (HQ / HK);
  z.row_tiles = (z.rows + 31) / 32;
  z.all_rows = shared ? z.rows * W : z.rows;
  z.all_tiles = (z.all_rows + 31) / 32;
  z.shared_groups = shared ? (int64_t)(B / W) * HK * z.all_tiles : 0;
  z.groups = z.shared_groups + (int64_t)B * HK * z.row_tiles;
  const int64_t all = ((int64_t)S + 31) / 32 + 1;  // the sinks' end and the window's begin may share one
  const int64_t seen = ((int64_t)sinks + 31) / 32 + ((int64_t)window + n + 61) / 32;
  z.tiles = z.shared_groups * (S / 32) + (z.groups - z.shared_groups) * (seen < all ? seen : all);
  z.units = cache_units(z.tiles, D);
  const int64_t live = z.all_rows < 32 ? z.all_rows : 32;
  z.floats = cache_ends_floats(z.groups) + (z.units + z.groups) * live * (D + 2);
  return z;
}

hipError_t launch_attn_paged(const AttnPagedArgs& a, const PagedSizes& z, int dt, int D, hipStream_t s,
                             bool* supported);

}  // namespace esep
