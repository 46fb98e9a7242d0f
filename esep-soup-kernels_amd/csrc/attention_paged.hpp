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
  bool shared;
  int solo;  // one launch: wavefronts to a block, else 0
};
// One launch, a block of four or eight wavefronts to a group, instead of the cut walk with its partials and their
// join: where one round of blocks takes all groups, and a block's wavefronts have only so many tiles more than the
// walk's would (up to four of few tiles; of many, 5 / 8 of an equal share, as rows are ragged) that its launch and,
// with many groups, their partials cost more. As many wavefronts as the rings of a CU's LDS allow: at D = 64 eight,
// while a CU has one block.
//
// Both launches / one in us (graph replays over caches that no cache of the card holds; *: taken, else the one
// launch). D = 128, 28 / 4 heads: 64 rows of up to 300 tokens 17.9 / 10.5, 1500 35.3 / 29.5, 2500 55.5 / 52.9, 4000
// 77.9* / 79.9; 32 of 700 17.5 / 14.0, 2000 26.5* / 29.5; 5 of 900 13.1 / 14.5 (the launch saved takes the host 3
// us); 12 / 2 heads, one row of 60 8.3 / 4.8, 700 9.3 / 11.6 (the same), 1000 9.5* / 14.6. D = 64, 14 / 2 heads, both
// / four wavefronts / eight: one row of 300 8.4 / 5.8 / 6.1, 700 9.1 / 8.2 / 7.2, 1500 9.5* / 12.6 / 10.1; 32 of 1000
// 14.1 / 11.5 / 10.7, 2500 17.2* / 20.6 / 19.1; 7 of 5 new tokens and a window of 1500 14.4 / 16.5 / 13.7; 120 of
// 4000 43.7 / 40.7 / 40.9; 130 (260 groups) of 1200 23.0 / 19.1, 2000 29.2* / 31.9; 8 / 8 heads, 40 of 1200 22.6 /
// 21.5, 2000 28.4* / 36.6.
inline int paged_solo(int64_t groups, int64_t tiles, int D) {
  const int64_t waves = kAttnCUs * (D == 128 ? 4 : 8), total = groups * tiles;
  const int each = D == 64 && groups <= kAttnCUs ? 8 : 4;
  const int64_t few = total / kAttnCUs < 4 ? total / kAttnCUs : 4, many = total * 5 / 8 / waves;
  const int64_t more = D == 64 ? 4 + groups / 64 : 6 + groups / 40;
  return groups <= waves / each && (tiles + each - 1) / each <= (few > many ? few : many) + more ? each : 0;
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
  z.shared = shared && z.solo == 0;
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
