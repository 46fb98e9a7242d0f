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
// One launch, a block of one to eight wavefronts to a group, instead of the cut walk with its partials and their
// join: where a block's wavefronts have only so many tiles more than the walk's would that its launch, its search for
// a wavefront's first group and, with many groups, their partials and starts cost more. That is up to four of few
// tiles; of many, 5 / 8 of an equal share, as rows are ragged (all of it for a single row's), in one round of blocks;
// then a few, more with more groups. As many wavefronts to a block as the rings of the CUs' LDS allow, so that one
// round takes all groups where it can. Shared tokens count once: the one launch reads them for each row.
//
// Both launches / one in us (graph replays over caches that no cache of the card holds; *: taken, else the one
// launch). D = 128, 28 / 4 heads: 64 rows of up to 300 tokens 17.9 / 10.5, 1500 35.3 / 29.5, 2500 55.5 / 52.9, 4000
// 77.9* / 79.9; 32 of 700 17.5 / 14.0, 2000 26.5* / 29.5; 5 of 900 13.1 / 14.5 (the launch saved takes the host 3
// us); 256 of 300 31.8 / 25.0, 3000 203* / 212; 600 of 300 68.0 / 55.2, 1500 226* / 226; 4 of 128 new tokens and 2000
// 62.9 / 45.9, one of 512 and 4000 135 / 92; 4 beams each, 64 of 500 24.9 / 13.0, 2000 32.6* / 34.6, 256 of 300 35.2
// / 24.2. 12 / 2 heads: one row of 60 8.3 / 4.8, 700 9.3 / 11.6 (as before), 1000 9.5* / 14.6; 300 of 60 22.1 / 7.5;
// 3000 of 60 80.5 / 37.9. 32 / 32 heads: 64 of 500 75.5 / 74.7, 1500 180* / 209.
//
// D = 64, 14 / 2 heads: one row of 300 8.4 / 6.1, 700 9.1 / 7.2, 1500 9.5* / 10.1; 32 of 1000 14.1 / 10.7, 2500 17.2*
// / 19.1; 7 of 5 new tokens and a window of 1500 14.4 / 13.7; 120 of 4000 43.7 / 40.9; 130 of 1200 23.0 / 19.1, 2000
// 29.2* / 31.9; 700 of 60 24.7 / 7.7, 1500 81.7* / 79.4; 8 beams each, 2000 of 100 116 / 20. (With four wavefronts
// where eight fit: one row of 700 8.2, 32 of 1000 11.5.)
//
// All of these have rows of a quarter to all of the longest, and the 5 / 8 is theirs. The rule sees the tables' width alone:
// where one row is that long and the others have 20 to 100 tokens, the one launch lasts as long as that row's block. One of 2500
// among 256, 28 / 4 heads of 128: 86.0 / 25.6 (in tables for 32768, which take the walk); of 2000 among 64 26.6 / 18.5;
// of 2800 among 1000, 14 / 2 heads of 64 69.8 / 32.8.
inline int paged_solo(int B, int64_t groups, int64_t tiles, int W, int D) {
  const int64_t waves = kAttnCUs * (D == 128 ? 4 : 8), total = groups * tiles / W;
  int each = D == 128 ? 4 : 8;
  while (each > 1 && groups * each > waves) each /= 2;
  const int64_t few = total / kAttnCUs < 4 ? total / kAttnCUs : 4;
  const int64_t many = groups > waves ? 0 : (B == 1 ? total : total * 5 / 8) / waves;
  const int64_t starts = groups < waves ? groups : waves;
  const int64_t more = D == 64 || W > 1 ? 4 + starts / 64 : 6 + starts / 40;
  return (tiles + each - 1) / each <= (few > many ? few : many) + more ? each : 0;
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
  z.solo = paged_solo(B, own, each, shared ? W : 1, D);
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
