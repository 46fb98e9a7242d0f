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
  bool shared, solo;
};
// One launch, a block of four wavefronts to a group, instead of the cut walk with its partials and their join: where one
// round of blocks takes all groups, and a block's wavefronts have only so many tiles more than the walk's would (up to
// four of few tiles; of many, 5 / 8 of an equal share, as rows are ragged) that its launch and, with many groups, their
// partials cost more. Both launches / one in us (graph replays), D = 128, 28 / 4 heads: 64 rows of up to 500 tokens 20.2 /
// 12.9, 1000 27.3 / 20.4, 2500 47.4 / 42.8, 4000 65.9* / 66.1; 32 of 2000 25.8* / 28.8, 5 of 900 12.8 / 13.3; 12 / 2 heads, one
// row of 60 8.8 / 5.3, 700 9.8 / 10.1 (the launch saved takes the host 3 us), 1000 10.1* / 12.6; 64 of up to 200 13.8 / 7.3;
// D = 64, 14 / 2 heads, 128 of up to 1500 23.1 / 17.1, 64 of 4096 26.0* / 29.2. (*: taken; else the one launch.)
constexpr int kPagedSoloWaves = 4;
inline bool paged_solo(int64_t groups, int64_t tiles, int D) {
  const int64_t waves = kAttnCUs * (D == 128 ? 4 : 8), total = groups * tiles;
  const int64_t few = total / kAttnCUs < 4 ? total / kAttnCUs : 4, many = total * 5 / 8 / waves;
  const int64_t more = 6 + groups / 40;
  return groups <= waves / kPagedSoloWaves && (tiles + 3) / kPagedSoloWaves <= (few > many ? few : many) + more;
}
inline PagedSizes paged_sizes(int B, int n, int W, int S, int HQ, int HK, int D, int window, int sinks,
                              bool shared) {
  PagedSizes z{};
  z.rows = (int64_t)n * (HQ / HK);
  z.row_tiles = (z.rows + 31) / 32;
  const int64_t own = (int64_t)B * HK * z.row_tiles;
  const int64_t all = ((int64_t)S + 31) / 32 + 1;  // the sinks' end and the window's begin may share one
  const int64_t seen = ((int64_t)sinks + 31) / 32 + ((int64_t)window + n + 61) / 32;
  const int64_t each = seen < all ? seen : all;
  z.solo = paged_solo(own, each, D);
  z.shared = shared && !z.solo;
  z.all_rows = z.shared ? z.rows * W : z.rows;
  z.all_tiles = (z.all_rows + 31) / 32;
  z.shared_groups = z.shared ? (int64_t)(B / W) * HK * z.all_tiles : 0;
  z.groups = z.shared_groups + own;
  z.tiles = z.shared_groups * (S / 32) + own * each;
  z.units = cache_units(z.tiles, D);
  const int64_t live = z.all_rows < 32 ? z.all_rows : 32;
  z.floats = z.solo ? 0 : cache_ends_floats(z.groups) + (z.units + z.groups) * live * (D + 2);
  return z;
}

hipError_t launch_attn_paged(const AttnPagedArgs& a, const PagedSizes& z, int dt, int D, hipStream_t s,
                             bool* supported);

}  // namespace esep
