// Attention of a row's n newest tokens over its cache (decoding: n = 1), with an optional window and sinks.
//
// Query t of a row sits at position len - n + t and sees key j <= that position, through a window only the last
// `window` of them and the first `sinks`. A kv head's query heads and new tokens make one tile of up to 32 query
// rows (row r: token r / G, head r % G of the group's G), so that K and V are read once for all of them, and a
// wavefront runs the causal kernels' 32-key step on it (attention_tiles.hpp): the matrix core is far from busy
// (512 of about 2000 cycles that a CU's share of the memory's rate leaves for a tile), so rows that do not
// fill the 32 cost nothing.
//
// Bound by the bytes of K and V, and below a few MB by the launches' latency. The 32-key tiles of all (row, kv
// head, query tile) groups are laid end to end and cut into equal runs, one to a wavefront, whatever the rows'
// lengths: the wavefronts end together. Each keeps a ring of two tiles in LDS for itself, filled by LDS
// DMA, and needs no barrier. A group within one run is stored; one that is cut leaves partials (maximum, sum
// and weighted sum in fp32, slot = wavefront + group) that k_attn_cache_join adds in their order.
//
// Kernel trace, walk + join: 32 rows of up to 8192 tokens, 28 / 4 heads of 128, bf16 56.9 + 4.6 us (334 MB, 5.4
// TB/s; a copy reaches 5.0, half of it writes); 8 rows of up to 32768 through a window of 4096, 12 / 2 heads 12.7
// + 3.9; one row of 700 tokens 6.0 + 3.8; 16 new tokens over 4 rows of up to 4001, 14 / 2 heads of 64 14.2 + 4.2.
#include <cmath>

#include "attention_cache.hpp"
#include "attention_tiles.hpp"

namespace esep {
namespace {

// Row b's keys for its n queries: `ns` tiles of the sinks from 0, then tiles from lo to len.
struct CacheRow {
  int len, lo, sink_hi, ns, tiles;
};
__device__ __forceinline__ CacheRow cache_row(const AttnCacheArgs& a, int b) {
  CacheRow r;
  const int len = a.len[b];
  r.len = len < 0 ? 0 : (len > a.S ? a.S : len);
  const int first = r.len > a.n ? r.len - a.n : 0;  // the first query's position
  r.sink_hi = a.sinks < r.len ? a.sinks : r.len;
  r.lo = first - a.window + 1;  // window >= 1
  if (r.lo <= r.sink_hi) r.lo = 0;
  r.ns = r.lo > 0 ? (r.sink_hi + 31) / 32 : 0;
  r.tiles = r.ns + (r.len - r.lo + 31) / 32;
  return r;
}

// The plan, and (found with the same reads where the rows are at most 64) the row whose tiles hold the first
// of wavefront u, with the number of that row's first tile; row -1: no work. per_tile: groups of a row.
template <int D>
__device__ __forceinline__ CachePlan cache_find(const AttnCacheArgs& a, int per_tile, int u, int* row,
                                                int* first) {
  const int lane = threadIdx.x & 63;
  auto tiles_of = [&](int b) { return b < a.B ? cache_row(a, b).tiles * per_tile : 0; };
  const int mine0 = tiles_of(lane);
  int sum = mine0;
  for (int b = lane + 64; b < a.B; b += 64) sum += tiles_of(b);
  const CachePlan p = cache_plan(lane_sum(sum), D);
  *row = -1;
  *first = 0;
  if (u >= p.units) return p;
  const int x = p.cut(u);
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int mine = b0 == 0 ? mine0 : tiles_of(b0 + lane);
    int run = mine;  // inclusive sums
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(run, d);
      if (lane >= d) run += o;
    }
    const uint64_t past = __ballot(before + run > x);
    if (past != 0) {
      const int l = (int)__builtin_ctzll(past);
      *row = b0 + l;
      *first = before + __builtin_amdgcn_readlane(run - mine, l);
      break;
    }
    before += __builtin_amdgcn_readlane(run, 63);
  }
  return p;
}

// One wavefront's fill of a 32-row swizzled tile (attention.hpp: SwzFill, whose row groups four wavefronts
// share).
template <int RB, bool NT>
struct CacheFill {
  static constexpr int GR = 1024 / RB, CH = RB / 16, N = 32 / GR, V = RB == 256 ? 4 : 2;
  int lrow, chunk;
  int64_t rs;  // bytes between tokens
  uint32_t voff[V];
  __device__ __forceinline__ CacheFill(int lane, int64_t rs_) : rs(rs_) {
    lrow = lane / CH;
    chunk = (lane % CH) ^ swz<RB>(lrow);
#pragma unroll
    for (int i = 0; i < V; ++i) voff[i] = (uint32_t)(lrow * rs) + 16u * (uint32_t)(chunk ^ i);
  }
  // rows r0 .. r0 + 31; those at or past rend repeat row rend - 1
  __device__ __forceinline__ void tile(char* dst, const char* base, int r0, int rend) const {
    if (r0 + 32 <= rend) {
#pragma unroll
      for (int q = 0; q < N; ++q)
        if constexpr (NT)
          lds_dma_x4_s_nt(base + (int64_t)(r0 + GR * q) * rs, voff[q % V], dst + 1024 * q);
        else
          lds_dma_x4_s(base + (int64_t)(r0 + GR * q) * rs, voff[q % V], dst + 1024 * q);
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q) {
        const int r = r0 + GR * q + lrow < rend ? r0 + GR * q + lrow : rend - 1;
        lds_dma_x4(base + (int64_t)r * rs + 16 * (chunk ^ (q % V)), dst + 1024 * q);
      }
    }
  }
};

// NT: K and V past the caches, where one query tile alone reads them, in rows of 256 bytes (32 rows of up to
// 8192 tokens, 28 / 4 heads: 69 -> 63 us; at D = 64 24 -> 25 for 64 rows of up to 4096, 14 / 2 heads).
template <typename T, int D, bool NT>
__global__ __launch_bounds__(64, D == 128 ? 2 : 3) void k_attn_cache(const AttnCacheArgs a) {
  constexpr int RB = 2 * D, TILE = 32 * RB;
  using V8 = typename Mfma<T>::v8;
  using Fill = CacheFill<RB, NT>;
  __shared__ __align__(1024) char kv[2][2][TILE];  // [buffer][K, V]

  const int lane = threadIdx.x, lq = lane & 31, hi = lane >> 5;
  const int G = a.HQ / a.HK, rows = G * a.n, RT = (rows + 31) / 32, per_tile = a.HK * RT;
  const int u = blockIdx.x;
  int first, b;
  const CachePlan plan = cache_find<D>(a, per_tile, u, &b, &first);
  if (b < 0) return;
  int x = plan.cut(u);
  const int x1 = plan.cut(u + 1);
  CacheRow row = cache_row(a, b);
  const Fill fk(lane, a.k_ts * (int64_t)sizeof(T)), fv(lane, a.v_ts * (int64_t)sizeof(T));
  const int live = rows < 32 ? rows : 32;  // rows of a partial

  while (x < x1) {
    while (x >= first + row.tiles * per_tile) {
      first += row.tiles * per_tile;
      row = cache_row(a, ++b);
    }
    const int gi = (x - first) / row.tiles;  // kv head and query tile within the row
    const int g0 = first + gi * row.tiles;
    const int t0 = x - g0, t1 = x1 - g0 < row.tiles ? x1 - g0 : row.tiles;
    const int kvh = gi / RT, rt = gi % RT;
    const char* kbase = reinterpret_cast<const char*>(
        static_cast<const T*>(a.k) + (int64_t)b * a.k_bs + (int64_t)kvh * a.k_hs);
    const char* vbase = reinterpret_cast<const char*>(
        static_cast<const T*>(a.v) + (int64_t)b * a.v_bs + (int64_t)kvh * a.v_hs);
    auto start_of = [&](int t) { return t < row.ns ? 32 * t : row.lo + 32 * (t - row.ns); };
    auto issue = [&](int t) {
      const int rend = t < row.ns ? row.sink_hi : row.len;
      fk.tile(kv[t & 1][0], kbase, start_of(t), rend);
      fv.tile(kv[t & 1][1], vbase, start_of(t), rend);
    };
    // every read of the ring by the group before is done
    __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
    issue(t0);
    if (t0 + 1 < t1) issue(t0 + 1);

    const int r = 32 * rt + lq, tok = r / G, h = kvh * G + r % G;
    const bool rok = r < rows;
    V8 qb[D / 16];
    {
      const T* qrow = static_cast<const T*>(a.q) + (int64_t)b * a.q_bs + (int64_t)tok * a.q_ts +
                      (int64_t)h * a.q_hs + 8 * hi;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) qb[c] = rok ? ld16<V8>(qrow + 16 * c) : V8{};
    }
    // positions: the lane's, and the tile's first and last
    const int p0 = row.len - a.n, pos = rok ? p0 + tok : p0 + a.n - 1;
    const int ufirst = p0 + 32 * rt / G;
    const int ulast = 32 * rt + 31 < rows ? p0 + (32 * rt + 31) / G : p0 + a.n - 1;
    f32x16 oacc[D / 32];
#pragma unroll
    for (int md = 0; md < D / 32; ++md) oacc[md] = f32x16{};
    float m = -INFINITY, l = 0.f;
    // q and the first tiles are here (through the builtin: the compiler then waits for no load of its own
    // within the loop, which would wait for the tile in flight too)
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    for (int t = t0; t < t1; ++t) {
      const int kh = start_of(t), cap = t < row.ns ? row.sink_hi - 1 : 0x7fffffff;
      const char* ks = kv[t & 1][0];
      const char* vs = kv[t & 1][1];
      fwd_tile_swz<T, D>(ks, vs, lane, a.scale_log2, qb, oacc, m, l,
                         [&](f32x16& acc) __attribute__((always_inline)) {
                           mask_window(acc, kh, ufirst < cap ? ufirst : cap, ulast - a.window,
                                       pos < cap ? pos : cap, pos - a.window, row.sink_hi, hi);
                         });
      // this tile's reads are done: its buffer takes tile t + 2; then tile t + 1 is waited for
      __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
      __builtin_amdgcn_sched_barrier(0);
      if (t + 2 < t1) {
        issue(t + 2);
        __builtin_amdgcn_s_waitcnt(wait_vm(2 * Fill::N));
      } else {
        __builtin_amdgcn_s_waitcnt(kWaitVm0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    x += t1 - t0;
    const int group = b * per_tile + gi;
    float* part = a.part + (int64_t)(u + group) * live * (D + 2);
    // the wavefront with a group's first tile says for the join which others have some
    if (t0 == 0 && lane == 0) a.ends[group] = make_int2(u, plan.unit_of(g0 + row.tiles - 1));
    if (rok && t0 == 0 && t1 == row.tiles) {  // the whole group
      store_rows_t<T, D>(static_cast<T*>(a.o) + (((int64_t)b * a.n + tok) * a.HQ + h) * D, oacc, hi,
                         l > 0.f ? 1.f / l : 0.f);
    } else if (rok) {
      if (hi == 0) {
        part[lq] = m;
        part[live + lq] = l;
      }
      float* po = part + 2 * live + lq * D + 4 * hi;
#pragma unroll
      for (int md = 0; md < D / 32; ++md)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
            *reinterpret_cast<float2*>(po + 32 * md + 8 * j + e) =
                make_float2(oacc[md][4 * j + e], oacc[md][4 * j + e + 1]);
    }
  }
}

// The groups that were cut, and zeros for the rows without tokens: one block per query row. A lane adds two
// columns over every GROUPS-th part with a running maximum, so that the parts are read once.
template <typename T, int D, int THREADS>
__global__ __launch_bounds__(THREADS) void k_attn_cache_join(const AttnCacheArgs a) {
  constexpr int PAIRS = D / 2, GROUPS = THREADS / PAIRS;
  __shared__ float2 sums[GROUPS][PAIRS];
  __shared__ float2 stat[GROUPS];  // maximum, sum
  const int G = a.HQ / a.HK, rows = G * a.n, RT = (rows + 31) / 32;
  const int rg = (int)(blockIdx.x % rows);
  const int kvh = (int)(blockIdx.x / rows % a.HK), b = (int)(blockIdx.x / rows / a.HK);
  const int group = (b * a.HK + kvh) * RT + rg / 32, lq = rg % 32, live = rows < 32 ? rows : 32;
  const int len = a.len[b];
  const int2 ends = a.ends[group];  // not written where the row has no token
  const int g = threadIdx.x / PAIRS, c = threadIdx.x % PAIRS;
  T* out = static_cast<T*>(a.o) + (((int64_t)b * a.n + rg / G) * a.HQ + kvh * G + rg % G) * D + 2 * c;
  if (len <= 0 || a.S <= 0) {
    if (g == 0) out[0] = out[1] = (T)0.f;
    return;
  }
  if (ends.x == ends.y) return;  // stored by its wavefront
  const int64_t size = (int64_t)live * (D + 2);
  const float* part = a.part + group * size;
  float m = -INFINITY, l = 0.f;
  float2 acc = make_float2(0.f, 0.f);
#pragma unroll 4
  for (int u = ends.x + g; u <= ends.y; u += GROUPS) {
    const float* p = part + u * size;
    const float pm = p[lq], pl = p[live + lq];
    const float2 v = *reinterpret_cast<const float2*>(p + 2 * live + lq * D + 2 * c);
    const float top = fmaxf(m, pm), ref = top == -INFINITY ? 0.f : top;
    const float w0 = exp2_fast(m - ref), w1 = exp2_fast(pm - ref);
    l = fmaf(w1, pl, w0 * l);
    acc.x = fmaf(w1, v.x, w0 * acc.x);
    acc.y = fmaf(w1, v.y, w0 * acc.y);
    m = top;
  }
  sums[g][c] = acc;
  if (c == 0) stat[g] = make_float2(m, l);
  __syncthreads();
  if (g != 0) return;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) top = fmaxf(top, stat[i].x);
  const float ref = top == -INFINITY ? 0.f : top;
  float den = 0.f;
  acc = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const float w = exp2_fast(stat[i].x - ref);
    den = fmaf(w, stat[i].y, den);
    acc.x = fmaf(w, sums[i][c].x, acc.x);
    acc.y = fmaf(w, sums[i][c].y, acc.y);
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  out[0] = (T)(acc.x * inv);
  out[1] = (T)(acc.y * inv);
}

template <typename T, int D>
hipError_t run(const AttnCacheArgs& a, hipStream_t s) {
  const int64_t units = cache_units(cache_tiles(a.B, a.n, a.S, a.HQ, a.HK, a.window, a.sinks), D);
  const dim3 grid((unsigned)(units > 0 ? units : 1)), rows((unsigned)(a.B * a.HQ * a.n));
  const bool once = D == 128 && cache_row_tiles(a.n, a.HQ, a.HK) == 1;
  if (once)
    hipLaunchKernelGGL((k_attn_cache<T, D, D == 128>), grid, dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((k_attn_cache<T, D, false>), grid, dim3(64), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (units > kCacheManyParts * cache_groups(a.B, a.n, a.HQ, a.HK) && rows.x <= 256)
    hipLaunchKernelGGL((k_attn_cache_join<T, D, 1024>), rows, dim3(1024), 0, s, a);
  else
    hipLaunchKernelGGL((k_attn_cache_join<T, D, 256>), rows, dim3(256), 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t run_d(const AttnCacheArgs& a, int D, hipStream_t s, bool* sup) {
  *sup = D == 128 || D == 64;
  if (D == 128) return run<T, 128>(a, s);
  if (D == 64) return run<T, 64>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_attn_cache(const AttnCacheArgs& a, int dt, int D, hipStream_t s, bool* sup) {
  if (dt == 1) return run_d<_Float16>(a, D, s, sup);
  if (dt == 2) return run_d<__bf16>(a, D, s, sup);
  *sup = false;
  return hipErrorInvalidValue;
}

}  // namespace esep
