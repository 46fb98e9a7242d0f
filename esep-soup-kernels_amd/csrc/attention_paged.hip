// Attention of a row's n newest tokens over its pages (decoding: n = 1), with an optional window and sinks: the walk
// of attention_cache.hip with the tokens' addresses found through a block table.
//
// Token j of row b lies in page tables[b, j / P] at place j % P. A tile of 32 keys begins at a multiple of 32, so
// that each half of it lies in one page (P is a power of two of at least 16). A wavefront reads the pages of 32 tiles
// at once, a half to a lane, and takes each tile's two from there. Keys before a window or past the length repeat the
// nearest one that is seen and are masked; what a page outside the pool should hold is not read: its keys are
// masked and its values count as 0.
//
// Rows whose first tokens lie in the same pages (the beams of a request) are walked together over those, their query
// rows in common tiles of 32: K and V of the shared tokens are read once for all of them. Each row's own tokens
// come in a walk of its own, and the join adds both.
//
// Bound by the bytes of K and V, and below a few MB by latency: where rows are short, one launch (k_attn_paged_solo) takes
// the walk's and the join's place (the rule and both sides' times: attention_paged.hpp).
//
// Kernel trace, walk + join: 48 rows of up to 8192 tokens, 28 / 4 heads of 128, bf16, pages of 64 85.8 + 4.8 us (497
// MB, 5.8 TB/s in the walk; a copy reaches 5.0, half of it writes); 8 requests of 4 beams over up to 8000 shared
// tokens and 130 each, pages of 16 29.8 + 7.0 (96 MB, and 13.9 MB of partials written, by the counter; each beam on its
// own 4 times the bytes of the prompt; 27.4 without the walk's products, 25.5 without its partials' stores). In one
// launch: 5 new tokens over 7 rows through a window of 1500, 14 / 2 heads of 64 14.4 (in two 12.6 + 4.0); one row of
// 700 tokens, 12 / 2 heads 9.7 (6.6 + 3.8). A CU of its own takes in up to 70 GB/s; a wavefront's products of a tile
// take 0.3 (D = 64) and 0.44 us (128). Tried in vain: rings of three and four tiles with fewer wavefronts (beams -4%,
// 256 rows of 300 tokens +20%), one to three tiles to a wavefront (-7% to +7% over twenty shapes), partials eight
// columns at a time (the join reads 32 bytes of a line) or through LDS in whole lines (no change over twenty shapes),
// joins by 512 threads (+1 to 4%) or of half the columns (-4 to +24%). Four wavefronts to a block whose tails meet in
// LDS, one partial for four, took 29.6 + 5.1 us at the beams and 10.2 instead of 7.0 in the walk of the one row; that row
// has had its own launch since, so that for shared pages this is open.
#include <cmath>

#include "attention_cache.hpp"
#include "attention_paged.hpp"
#include "attention_paged_tiles.hpp"

namespace esep {
namespace {

__device__ __forceinline__ int paged_len(const AttnPagedArgs& a, int b) {
  const int len = a.len[b], S = a.tokens();
  return len < 0 ? 0 : (len > S ? S : len);
}
// Tokens of the W rows from r W on that are walked together: whole tiles, all of them seen by every new token.
__device__ __forceinline__ int shared_len(const AttnPagedArgs& a, int r) {
  int s = a.shared[r];
  for (int w = 0; w < a.W; ++w) {
    const int most = paged_len(a, r * a.W + w) - a.n;
    s = s < most ? s : most;
  }
  return s > 0 ? s & ~31 : 0;
}

// Rows that are walked together: keys lo .. len in tiles from a multiple of 32 on, before them `ns` tiles of the sinks.
struct PagedRow {
  int b, len, lo, sink_hi, ns, tiles;
  bool common;  // W rows from b on, over what they share
  int shared;   // tokens of the row's keys that a common walk takes
};
template <bool SHARED>
__device__ __forceinline__ PagedRow paged_row(const AttnPagedArgs& a, int e) {
  PagedRow r{};
  if constexpr (SHARED) {
    const int R = a.B / a.W;
    if (e < R) {
      r.common = true;
      r.b = e * a.W;
      r.len = shared_len(a, e);
      r.tiles = r.len / 32;
      return r;
    }
    r.b = e - R;
    r.shared = r.lo = shared_len(a, r.b / a.W);
    r.len = paged_len(a, r.b);
  } else {
    r.b = e;
    r.len = paged_len(a, e);
    const int first = r.len > a.n ? r.len - a.n : 0;  // the first query's position
    r.sink_hi = a.sinks < r.len ? a.sinks : r.len;
    r.lo = first - a.window + 1;  // window >= 1
    if (r.lo <= r.sink_hi) r.lo = 0;
    r.ns = r.lo > 0 ? (r.sink_hi + 31) / 32 : 0;
  }
  r.tiles = r.ns + (r.len - (r.lo & ~31) + 31) / 32;
  return r;
}

// The plan, and the place (rows e) whose tiles hold the first of wavefront u, with the number of that place's first
// tile; place -1: no work.
template <int D, bool SHARED>
__device__ __forceinline__ CachePlan paged_find(const AttnPagedArgs& a, int per, int per_common, int u, int* place,
                                                int* first) {
  const int lane = threadIdx.x & 63, R = SHARED ? a.B / a.W : 0, E = a.B + R;
  auto tiles_of = [&](int e) {
    return e < E ? paged_row<SHARED>(a, e).tiles * (e < R ? per_common : per) : 0;
  };
  const int mine0 = tiles_of(lane);
  int sum = mine0;
  for (int e = lane + 64; e < E; e += 64) sum += tiles_of(e);
  const CachePlan p = cache_plan(lane_sum(sum), D);
  *place = -1;
  *first = 0;
  if (u >= p.units) return p;
  const int x = p.cut(u);
  int before = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int mine = e0 == 0 ? mine0 : tiles_of(e0 + lane);
    int run = mine;  // inclusive sums
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(run, d);
      if (lane >= d) run += o;
    }
    const uint64_t past = __ballot(before + run > x);
    if (past != 0) {
      const int l = (int)__builtin_ctzll(past);
      *place = e0 + l;
      *first = before + __builtin_amdgcn_readlane(run - mine, l);
      break;
    }
    before += __builtin_amdgcn_readlane(run, 63);
  }
  return p;
}

// One wavefront's fill of a 32-row swizzled tile from two runs of 16 tokens.
template <int RB, bool NT>
struct PagedFill {
  static constexpr int GR = 1024 / RB, CH = RB / 16, N = 32 / GR, V = RB == 256 ? 4 : 2;
  int lrow, chunk;
  int64_t ps, ts;  // bytes between pages, tokens
  int mask;        // P - 1
  uint32_t voff[V];
  __device__ __forceinline__ PagedFill(int lane, int64_t ps_, int64_t ts_, int mask_) : ps(ps_), ts(ts_), mask(mask_) {
    lrow = lane / CH;
    chunk = (lane % CH) ^ swz<RB>(lrow);
#pragma unroll
    for (int i = 0; i < V; ++i) voff[i] = (uint32_t)(lrow * ts) + 16u * (uint32_t)(chunk ^ i);
  }
  // keys k0 .. k0 + 31, all of them there: the halves in pages g0 and g1
  __device__ __forceinline__ void whole(char* dst, const char* base, int k0, int g0, int g1) const {
    const char* h[2] = {base + g0 * ps + (k0 & mask) * ts, base + g1 * ps + ((k0 + 16) & mask) * ts};
#pragma unroll
    for (int q = 0; q < N; ++q) {
      const char* at = h[q / (N / 2)] + GR * (q % (N / 2)) * ts;
      if constexpr (NT)
        lds_dma_x4_s_nt(at, voff[q % V], dst + 1024 * q);
      else
        lds_dma_x4_s(at, voff[q % V], dst + 1024 * q);
    }
  }
  // the lane's key of row group q, within lo .. hi - 1, and where it lies
  __device__ __forceinline__ const char* at(const char* base, int q, int k0, int lo, int hi, int g0, int g1,
                                            int* page) const {
    int k = k0 + GR * q + lrow;
    k = k < lo ? lo : (k < hi ? k : hi - 1);
    *page = k - k0 < 16 ? g0 : g1;
    return base + *page * ps + (k & mask) * ts + 16 * (chunk ^ (q % V));
  }
  __device__ __forceinline__ void partial(char* dst, const char* base, int k0, int lo, int hi, int g0, int g1) const {
#pragma unroll
    for (int q = 0; q < N; ++q) {
      int page;
      lds_dma_x4(at(base, q, k0, lo, hi, g0, g1, &page), dst + 1024 * q);
    }
  }
  // the same where a page may be none of the n: zeros for its keys
  __device__ __forceinline__ void checked(char* dst, const char* base, int k0, int lo, int hi, int g0, int g1, int n,
                                          int lane) const {
    for (int q = 0; q < N; ++q) {
      int page;
      const char* p = at(base, q, k0, lo, hi, g0, g1, &page);
      uint4 x = make_uint4(0, 0, 0, 0);
      if ((unsigned)page < (unsigned)n) x = *reinterpret_cast<const uint4*>(p);
      *reinterpret_cast<uint4*>(dst + 1024 * q + 16 * lane) = x;
    }
  }
};

// Query row r of a kv head's `rows`: its batch row, token and head.
struct PagedQuery {
  int G, rows, b, tok, h;
  bool ok;
  __device__ __forceinline__ PagedQuery(const AttnPagedArgs& a, const PagedRow& row, int kvh, int r) {
    G = a.HQ / a.HK;
    const int own = G * a.n;
    rows = row.common ? a.W * own : own;
    ok = r < rows;
    const int q = ok ? r : 0;
    b = row.b + q / own;
    tok = q % own / G;
    h = kvh * G + q % G;
  }
};

// A wavefront's tiles t0 .. t1 - 1 of one group through its own ring into `x`, its query rows (tile rt of the kv head's).
template <typename T, int D, bool NT, int ROWS>
__device__ __forceinline__ void paged_walk(const AttnPagedArgs& a, const PagedRow& row, const PagedQuery& at, int kvh,
                                           int rt, int t0, int t1, const PagedFill<2 * D, NT>& fk,
                                           const PagedFill<2 * D, NT>& fv, char (&kv)[2][2][32 * 2 * D], int lane,
                                           PagedTile<T, D, ROWS>& x) {
  using Fill = PagedFill<2 * D, NT>;
  const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + (int64_t)kvh * a.k_hs);
  const char* vbase = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + (int64_t)kvh * a.v_hs);
  const int32_t* table = a.tables + (int64_t)row.b * a.t_bs;
  const int lo0 = row.lo & ~31;
  auto start_of = [&](int t) { return t < row.ns ? 32 * t : lo0 + 32 * (t - row.ns); };
  int ids = -1, ids0 = 0;  // lane l: the page of half l % 2 of tile ids0 + l / 2
  auto load_ids = [&](int t) {
    ids0 = t;
    const int tl = t + lane / 2;
    ids = -1;
    if (tl < t1) {
      const int from = tl < row.ns ? 0 : row.lo, to = tl < row.ns ? row.sink_hi : row.len;
      int k = start_of(tl) + 16 * (lane & 1);
      k = k < from ? from : (k < to ? k : to - 1);
      ids = table[k >> a.page_shift];
    }
    asm volatile("" : "+v"(ids));  // here now: a wait for it in the loop would wait for the tiles in flight too
  };
  uint32_t bad = 0;  // bits 2 buffer + half: the page is none
  // asks for tile t; false: it is there already, without a DMA
  auto issue = [&](int t) {
    if (t - ids0 >= 32) load_ids(t);
    const int p0 = __builtin_amdgcn_readlane(ids, 2 * (t - ids0));
    const int p1 = __builtin_amdgcn_readlane(ids, 2 * (t - ids0) + 1);
    const int k0 = start_of(t), from = t < row.ns ? 0 : row.lo, to = t < row.ns ? row.sink_hi : row.len;
    char* kd = kv[t & 1][0];
    char* vd = kv[t & 1][1];
    const uint32_t none = ((unsigned)p0 >= (unsigned)a.N ? 1u : 0u) | ((unsigned)p1 >= (unsigned)a.N ? 2u : 0u);
    bad = (bad & ~(3u << (2 * (t & 1)))) | none << (2 * (t & 1));
    if (none) {
      fk.checked(kd, kbase, k0, from, to, p0, p1, a.N, lane);
      fv.checked(vd, vbase, k0, from, to, p0, p1, a.N, lane);
      return false;
    }
    if (k0 >= from && k0 + 32 <= to) {
      fk.whole(kd, kbase, k0, p0, p1);
      fv.whole(vd, vbase, k0, p0, p1);
    } else {
      fk.partial(kd, kbase, k0, from, to, p0, p1);
      fv.partial(vd, vbase, k0, from, to, p0, p1);
    }
    return true;
  };
  // every read of the ring by the group before is done
  __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
  load_ids(t0);
  issue(t0);
  if (t0 + 1 < t1) issue(t0 + 1);

  x.load(static_cast<const T*>(a.q) + (int64_t)at.b * a.q_bs + (int64_t)at.tok * a.q_ts + (int64_t)at.h * a.q_hs, at.ok);
  // positions: the lane's, and the tile's first and last
  const int p0 = row.len - a.n, pos = at.ok ? p0 + at.tok : p0 + a.n - 1;
  const int ufirst = p0 + ROWS * rt / at.G;
  const int ulast = ROWS * (rt + 1) <= at.rows ? p0 + (ROWS * (rt + 1) - 1) / at.G : p0 + a.n - 1;
  // q and the first tiles are here (through the builtin: the compiler then waits for no load of its own
  // within the loop, which would wait for the tile in flight too)
  __builtin_amdgcn_s_waitcnt(kWaitVm0);
  for (int t = t0; t < t1; ++t) {
    // a window's tiles have no sinks (the first of them may begin among those)
    const int kh = start_of(t), cap = t < row.ns ? row.sink_hi - 1 : 0x7fffffff;
    const int sinks = t < row.ns || row.lo == 0 ? row.sink_hi : 0;
    const int top = pos < cap ? pos : cap, low = pos - a.window;
    const bool some = !row.common && (kh + 31 > (ufirst < cap ? ufirst : cap) || kh <= ulast - a.window);
    x.step(kv[t & 1][0], kv[t & 1][1], a.scale_log2, kh, some, bad >> (2 * (t & 1)) & 3,
           [&](int key) { return key > top || (key <= low && key >= sinks); });
    // this tile's reads are done: its buffer takes tile t + 2; then tile t + 1 is waited for
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    __builtin_amdgcn_sched_barrier(0);
    if (t + 2 < t1 && issue(t + 2))
      __builtin_amdgcn_s_waitcnt(wait_vm(2 * Fill::N));
    else
      __builtin_amdgcn_s_waitcnt(kWaitVm0);
    __builtin_amdgcn_sched_barrier(0);
  }
  x.finish();
}

template <typename T, int D, bool NT, bool SHARED, int ROWS>
__global__ __launch_bounds__(64, D == 128 ? 2 : 3) void k_attn_paged(const AttnPagedArgs a) {
  constexpr int RB = 2 * D, TILE = 32 * RB;
  using Fill = PagedFill<RB, NT>;
  __shared__ __align__(1024) char kv[2][2][TILE];  // [buffer][K, V]

  const int lane = threadIdx.x;
  const int G = a.HQ / a.HK, own_rows = G * a.n, all_rows = SHARED ? a.W * own_rows : own_rows;
  const int per = a.HK * ((own_rows + 31) / 32), per_common = a.HK * ((all_rows + 31) / 32);
  const int R = SHARED ? a.B / a.W : 0;
  const int u = blockIdx.x;
  int first, e;
  const CachePlan plan = paged_find<D, SHARED>(a, per, per_common, u, &e, &first);
  if (e < 0) return;
  int x = plan.cut(u);
  const int x1 = plan.cut(u + 1);
  PagedRow row = paged_row<SHARED>(a, e);
  const int mask = (1 << a.page_shift) - 1;
  const Fill fk(lane, a.k_ps * (int64_t)sizeof(T), a.k_ts * (int64_t)sizeof(T), mask);
  const Fill fv(lane, a.v_ps * (int64_t)sizeof(T), a.v_ts * (int64_t)sizeof(T), mask);
  const int live = all_rows < 32 ? all_rows : 32;  // rows of a partial

  while (x < x1) {
    int here = e < R ? per_common : per;
    while (x >= first + row.tiles * here) {
      first += row.tiles * here;
      row = paged_row<SHARED>(a, ++e);
      here = e < R ? per_common : per;
    }
    const int RT = here / a.HK;
    const int gi = (x - first) / row.tiles;  // kv head and query tile
    const int g0 = first + gi * row.tiles;
    const int t0 = x - g0, t1 = x1 - g0 < row.tiles ? x1 - g0 : row.tiles;
    const int kvh = gi / RT, rt = gi % RT;
    PagedTile<T, D, ROWS> tile(lane);
    const PagedQuery at(a, row, kvh, ROWS * rt + tile.row());
    paged_walk<T, D, NT, ROWS>(a, row, at, kvh, rt, t0, t1, fk, fv, kv, lane, tile);
    x += t1 - t0;
    const int group = (e < R ? e * per_common : R * per_common + (e - R) * per) + gi;
    float* part = a.part + (int64_t)(u + group) * live * (D + 2);
    // the wavefront with a group's first tile says for the join which others have some
    if (t0 == 0 && lane == 0) a.ends[group] = make_int2(u, plan.unit_of(g0 + row.tiles - 1));
    if (at.ok && t0 == 0 && t1 == row.tiles && !(SHARED && (row.common || row.shared > 0))) {  // all of the row's keys
      tile.store(static_cast<T*>(a.o) + (((int64_t)at.b * a.n + at.tok) * a.HQ + at.h) * D);
    } else if (at.ok) {
      const int q = tile.row();
      if (tile.first()) {
        part[q] = tile.m;
        part[live + q] = tile.l;
      }
      float* sums = part + 2 * live + q * D;  // at even addresses
      tile.each4([&](int column, f32x4 v) {
        *reinterpret_cast<float2*>(sums + column) = make_float2(v[0], v[1]);
        *reinterpret_cast<float2*>(sums + column + 2) = make_float2(v[2], v[3]);
      });
    }
  }
}

// One launch for short rows: a block of NW wavefronts to a group, an equal share of its tiles to each, whose sums meet in
// LDS.
template <typename T, int D, int NW, bool NT, int ROWS>
__global__ __launch_bounds__(64 * NW, D == 128 ? 2 : 3) void k_attn_paged_solo(const AttnPagedArgs a) {
  constexpr int RB = 2 * D, TILE = 32 * RB;
  constexpr int LD = D + 4;  // floats of a row of sums: the 16-byte pieces of 32 rows on different banks
  static_assert(4 * TILE >= 32 * LD * 4, "the sums fit a ring");
  // [wavefront][buffer][K, V]. (Of a size known at launch only: told that a wavefront has a SIMD for itself, the compiler
  // keeps the accumulators in the other half of the registers and moves them back and forth.)
  extern __shared__ __align__(1024) char lds[];
  auto& rings = *reinterpret_cast<char (*)[NW][2][2][TILE]>(lds);
  __shared__ float stat[NW][2][32];  // maximum, sum
  const int lane = threadIdx.x & 63, w = wave_id();
  const int G = a.HQ / a.HK, RT = (G * a.n + 31) / 32;
  const int rt = (int)(blockIdx.x % RT), kvh = (int)(blockIdx.x / RT % a.HK), b = (int)(blockIdx.x / RT / a.HK);
  const PagedRow row = paged_row<false>(a, b);
  if constexpr (NW == 1) {
    const int mask = (1 << a.page_shift) - 1;
    const PagedFill<RB, NT> fk(lane, a.k_ps * (int64_t)sizeof(T), a.k_ts * (int64_t)sizeof(T), mask);
    const PagedFill<RB, NT> fv(lane, a.v_ps * (int64_t)sizeof(T), a.v_ts * (int64_t)sizeof(T), mask);
    PagedTile<T, D, ROWS> tile(lane);
    const PagedQuery at(a, row, kvh, ROWS * rt + tile.row());
    if (row.tiles > 0)
      paged_walk<T, D, NT, ROWS>(a, row, at, kvh, rt, 0, row.tiles, fk, fv, rings[0], lane, tile);
    else
      tile.load(nullptr, false);
    if (at.ok) tile.store(static_cast<T*>(a.o) + (((int64_t)at.b * a.n + at.tok) * a.HQ + at.h) * D);
    return;
  }
  const int each = (row.tiles + NW - 1) / NW, busy = each > 0 ? (row.tiles + each - 1) / each : 0;
  if (w < busy) {
    const int mask = (1 << a.page_shift) - 1;
    const PagedFill<RB, NT> fk(lane, a.k_ps * (int64_t)sizeof(T), a.k_ts * (int64_t)sizeof(T), mask);
    const PagedFill<RB, NT> fv(lane, a.v_ps * (int64_t)sizeof(T), a.v_ts * (int64_t)sizeof(T), mask);
    PagedTile<T, D, ROWS> tile(lane);
    const PagedQuery at(a, row, kvh, ROWS * rt + tile.row());
    const int t0 = w * each, t1 = t0 + each < row.tiles ? t0 + each : row.tiles;
    paged_walk<T, D, NT, ROWS>(a, row, at, kvh, rt, t0, t1, fk, fv, rings[w], lane, tile);
    float* sums = reinterpret_cast<float*>(rings[w]) + tile.row() * LD;
    tile.each4([&](int column, f32x4 v) { *reinterpret_cast<f32x4*>(sums + column) = v; });
    if (tile.first()) {
      stat[w][0][tile.row()] = tile.m;
      stat[w][1][tile.row()] = tile.l;
    }
  }
  __syncthreads();
  // lane q: the weights of row q's sums
  float top = -INFINITY, den = 0.f, f[NW];
#pragma unroll
  for (int c = 0; c < NW; ++c) {
    f[c] = c < busy ? stat[c][0][lane % ROWS] : -INFINITY;
    top = fmaxf(top, f[c]);
  }
  const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int c = 0; c < NW; ++c) {
    f[c] = exp2_fast(f[c] - ref);
    if (c < busy) den = fmaf(f[c], stat[c][1][lane % ROWS], den);
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  constexpr int C = D / 64, Q = 2;  // columns of a lane, rows at once
  typedef T Out __attribute__((ext_vector_type(C)));
  const int rows = G * a.n - ROWS * rt, most = rows < ROWS ? rows : ROWS;
  for (int q0 = w; q0 < most; q0 += Q * NW) {
    float acc[Q][C] = {};
#pragma unroll
    for (int c = 0; c < NW; ++c) {
      if (c >= busy) break;
      const float* v = reinterpret_cast<const float*>(rings[c]) + C * lane;
#pragma unroll
      for (int k = 0; k < Q; ++k) {
        const int q = q0 + k * NW < ROWS ? q0 + k * NW : ROWS - 1;
        const float fq = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f[c]), q));
#pragma unroll
        for (int i = 0; i < C; ++i) acc[k][i] = fmaf(fq, v[q * LD + i], acc[k][i]);
      }
    }
#pragma unroll
    for (int k = 0; k < Q; ++k) {
      const int q = q0 + k * NW, r = ROWS * rt + q;
      if (q >= most) break;
      const float iq = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(inv), q));
      Out out;
#pragma unroll
      for (int i = 0; i < C; ++i) out[i] = (T)(acc[k][i] * iq);
      *reinterpret_cast<Out*>(static_cast<T*>(a.o) +
                              (((int64_t)b * a.n + r / G) * a.HQ + kvh * G + r % G) * D + C * lane) = out;
    }
  }
}

// The groups that were cut or share keys, and zeros for the rows without tokens. A lane adds two columns of a query row
// over every GROUPS-th part with a running maximum, so that the parts are read once; a block has as many rows as
// its threads hold.
template <typename T, int D, int THREADS, int GROUPS, bool SHARED>
__global__ __launch_bounds__(THREADS) void k_attn_paged_join(const AttnPagedArgs a) {
  constexpr int PAIRS = D / 2, ROWS = THREADS / PAIRS / GROUPS;
  static_assert(ROWS == 1 || GROUPS == 1, "rows of a block do not wait for each other");
  __shared__ float2 sums[GROUPS][PAIRS];
  __shared__ float2 stat[GROUPS];  // maximum, sum
  const int G = a.HQ / a.HK, rows = G * a.n, all_rows = SHARED ? a.W * rows : rows;
  const int RT = (rows + 31) / 32, CT = (all_rows + 31) / 32, live = all_rows < 32 ? all_rows : 32;
  const int g = ROWS > 1 ? 0 : threadIdx.x / PAIRS, c = threadIdx.x % PAIRS;
  const int row = ROWS > 1 ? (int)(blockIdx.x * ROWS + threadIdx.x / PAIRS) : (int)blockIdx.x;
  if (ROWS > 1 && row >= a.B * a.HK * rows) return;
  const int rg = row % rows, kvh = row / rows % a.HK, b = row / rows / a.HK;
  T* out = static_cast<T*>(a.o) + (((int64_t)b * a.n + rg / G) * a.HQ + kvh * G + rg % G) * D + 2 * c;
  if (paged_len(a, b) <= 0) {
    if (g == 0) out[0] = out[1] = (T)0.f;
    return;
  }
  const int R = SHARED ? a.B / a.W : 0;
  const int own = R * a.HK * CT + (b * a.HK + kvh) * RT + rg / 32;
  const int2 ends = a.ends[own];
  int n = ends.y - ends.x + 1, common = 0, rc = 0;
  int2 more = make_int2(0, -1);
  if (SHARED && shared_len(a, b / a.W) > 0) {
    rc = b % a.W * rows + rg;
    common = (b / a.W * a.HK + kvh) * CT + rc / 32;
    more = a.ends[common];
  } else if (n == 1) {
    return;  // stored by its wavefront
  }
  const int own_parts = n;
  n += more.y - more.x + 1;
  const int64_t size = (int64_t)live * (D + 2);
  float m = -INFINITY, l = 0.f;
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int i = g; i < n; i += GROUPS) {
    const bool mine = i < own_parts;
    const int slot = mine ? ends.x + i + own : more.x + (i - own_parts) + common;
    const int lq = mine ? rg % 32 : rc % 32;
    const float* p = a.part + slot * size;
    const float pm = p[lq], pl = p[live + lq];
    const float2 v = *reinterpret_cast<const float2*>(p + 2 * live + lq * D + 2 * c);
    const float top = fmaxf(m, pm), ref = top == -INFINITY ? 0.f : top;
    const float w0 = exp2_fast(m - ref), w1 = exp2_fast(pm - ref);
    l = fmaf(w1, pl, w0 * l);
    acc.x = fmaf(w1, v.x, w0 * acc.x);
    acc.y = fmaf(w1, v.y, w0 * acc.y);
    m = top;
  }
  if constexpr (GROUPS > 1) {
    sums[g][c] = acc;
    if (c == 0) stat[g] = make_float2(m, l);
    __syncthreads();
    if (g != 0) return;
    m = -INFINITY;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) m = fmaxf(m, stat[i].x);
    const float ref = m == -INFINITY ? 0.f : m;
    l = 0.f;
    acc = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
      const float w = exp2_fast(stat[i].x - ref);
      l = fmaf(w, stat[i].y, l);
      acc.x = fmaf(w, sums[i][c].x, acc.x);
      acc.y = fmaf(w, sums[i][c].y, acc.y);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  out[0] = (T)(acc.x * inv);
  out[1] = (T)(acc.y * inv);
}

// Wavefronts to a group up to which a row's few parts are added by one lane each, so that a block joins 256 / (D / 2)
// rows (256 rows of up to 300 tokens in wider tables, 28 / 4 heads of 128: 38 -> 32 us in all; with it up to 8 wavefronts to a group
// 32 rows of 4 beams over up to 8000 shared tokens 35.3 -> 38.5).
constexpr int64_t kPagedFewParts = 2;

template <typename T, int D, int NW, int ROWS>
void solo(const AttnPagedArgs& a, const PagedSizes& z, hipStream_t s) {
  const dim3 grid((unsigned)z.groups), block(64 * NW);
  constexpr unsigned lds = NW * 4 * 32 * 2 * D;
  if (D == 128 && z.row_tiles == 1)
    hipLaunchKernelGGL((k_attn_paged_solo<T, D, NW, D == 128, ROWS>), grid, block, lds, s, a);
  else
    hipLaunchKernelGGL((k_attn_paged_solo<T, D, NW, false, ROWS>), grid, block, lds, s, a);
}

template <typename T, int D, bool SHARED, int ROWS>
void walk(const AttnPagedArgs& a, const PagedSizes& z, hipStream_t s) {
  if constexpr (!SHARED) {
    if constexpr (D == 64)
      if (z.solo == 8) return solo<T, D, 8, ROWS>(a, z, s);
    if (z.solo == 4) return solo<T, D, 4, ROWS>(a, z, s);
    if (z.solo == 2) return solo<T, D, 2, ROWS>(a, z, s);
    if (z.solo == 1) return solo<T, D, 1, ROWS>(a, z, s);
  }
  const dim3 grid((unsigned)(z.units > 0 ? z.units : 1));
  if (D == 128 && z.all_tiles == 1)
    hipLaunchKernelGGL((k_attn_paged<T, D, D == 128, SHARED, ROWS>), grid, dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((k_attn_paged<T, D, false, SHARED, ROWS>), grid, dim3(64), 0, s, a);
}

template <typename T, int D, bool SHARED>
hipError_t run(const AttnPagedArgs& a, const PagedSizes& z, hipStream_t s) {
  if (z.all_rows <= 16)
    walk<T, D, SHARED, 16>(a, z, s);
  else
    walk<T, D, SHARED, 32>(a, z, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || z.solo) return e;
  const unsigned rows = (unsigned)(a.B * a.HQ * a.n);
  constexpr unsigned per = 256 / (D / 2);
  if (z.units > kCacheManyParts * z.groups && rows <= 256)
    hipLaunchKernelGGL((k_attn_paged_join<T, D, 1024, 2048 / D, SHARED>), dim3(rows), dim3(1024), 0, s, a);
  else if (z.units > kPagedFewParts * z.groups)
    hipLaunchKernelGGL((k_attn_paged_join<T, D, 256, 512 / D, SHARED>), dim3(rows), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((k_attn_paged_join<T, D, 256, 1, SHARED>), dim3((rows + per - 1) / per), dim3(256), 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t run_d(const AttnPagedArgs& a, const PagedSizes& z, int D, hipStream_t s, bool* sup) {
  *sup = D == 128 || D == 64;
  if (D == 128) return a.shared ? run<T, 128, true>(a, z, s) : run<T, 128, false>(a, z, s);
  if (D == 64) return a.shared ? run<T, 64, true>(a, z, s) : run<T, 64, false>(a, z, s);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_attn_paged(const AttnPagedArgs& a, const PagedSizes& z, int dt, int D, hipStream_t s, bool* sup) {
  if (dt == 1) return run_d<_Float16>(a, z, D, s, sup);
  if (dt == 2) return run_d<__bf16>(a, z, D, s, sup);
  *sup = false;
  return hipErrorInvalidValue;
}

}  // namespace esep
