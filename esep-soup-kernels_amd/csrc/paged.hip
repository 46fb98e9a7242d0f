// The upkeep of paged caches: which page and place each new token gets (k_page_tables), the store of its key and
// value there (k_page_store), and the beams' states following their parents (k_beam_reorder).
#include "paged.hpp"

#include "common.hpp"

namespace esep {
namespace {

// ---------------------------------------------------------------------------------------
// Block tables and slots. Row b holds L_b tokens in ceil(L_b / P) pages and gets n_b more. Of its pages each begins
// with a token t, t % P = 0, so that a new page belongs to exactly one new token: page j of row b is entry
// taken + sum over the rows before of their new pages + j - ceil(L_b / P) of the free list. The work is laid out
// by tokens: a block takes kTableTokens of them, finds its rows by prefix sums over the rows (of n and of the new
// pages), 256 rows at a time, and a token its row by a binary search of those. Block 0 goes through all rows
// and writes the offsets and the new lengths.
//
// Bound by latency: lengths, a scan's two barriers, a page's number, the slot. 64 rows of one new token 3.5 us, 300 rows of up
// to 2047 (300000 tokens) 7.8, 4000 rows of one 22.6; a thread's four tokens ask for their pages together.
// ---------------------------------------------------------------------------------------
constexpr int kTableTokens = 1024, kTableEach = kTableTokens / 256;

__device__ __forceinline__ int pages_of(int64_t tokens, int P) { return (int)((tokens + P - 1) / P); }

// Inclusive sums of (x, y) over the block's 256 threads; *tx, *ty: the block's sums. Two barriers.
__device__ __forceinline__ void block_scan2(int64_t& x, int& y, int64_t* tx, int* ty, int64_t (&wx)[4], int (&wy)[4]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t ox = __shfl_up(x, d);
    const int oy = __shfl_up(y, d);
    if (lane >= d) x += ox, y += oy;
  }
  __syncthreads();
  if (lane == 63) wx[w] = x, wy[w] = y;
  __syncthreads();
  *tx = 0;
  *ty = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < w) x += wx[i], y += wy[i];
    *tx += wx[i];
    *ty += wy[i];
  }
}

// The block's tokens i0 .. i1; with `last` all rows are gone through and their offsets written, with `state` also
// the new lengths and the pages taken. Tokens past `total` are not added: the row that reaches it gets fewer, the rows
// behind it none.
__device__ void page_tables(const PageTablesArgs& a, int64_t i0, int64_t i1, bool last, bool state) {
  __shared__ int64_t wx[4];
  __shared__ int wy[4];
  __shared__ int r_end[256], r_len[256], r_held[256], r_first[256];  // r_end: tokens up to the row's last
  const int tid = threadIdx.x;
  const int64_t cap = (int64_t)a.M * a.P;
  const int64_t taken = *a.taken < 0 ? 0 : *a.taken;
  int64_t before = 0, pages = 0;  // tokens and new pages of the rows before these 256
  for (int b0 = 0; b0 < a.B; b0 += 256) {
    const int b = b0 + tid;
    int len = 0, add = 0;
    if (b < a.B) {
      len = a.lengths[b];
      len = len < 0 ? 0 : (len > cap ? (int)cap : len);
      add = a.add[b] < 0 ? 0 : a.add[b];
    }
    auto after = [&](int64_t n) { return len + n < cap ? len + n : cap; };
    const int held = pages_of(len, a.P), take = pages_of(after(add), a.P) - held;
    int64_t end = add, all;
    int upto = take, took;
    block_scan2(end, upto, &all, &took, wx, wy);
    end += before;
    const int64_t lo = end - add < a.total ? end - add : a.total, hi = end < a.total ? end : a.total;
    const int64_t first = taken + pages + (upto - take);  // the row's first new page in the free list
    r_end[tid] = (int)hi;
    r_len[tid] = len;
    r_held[tid] = held;
    r_first[tid] = first > 0x7fffffff ? 0x7fffffff : (int)first;
    if (last && b < a.B) {
      a.cu[b + 1] = (int)hi;
      if (state) {
        a.lengths_out[b] = (int)after(hi - lo);
        // the row that reaches `total` says what is taken
        if (lo < a.total && end >= a.total) {
          const int64_t now = first + pages_of(after(hi - lo), a.P) - held;
          *a.taken_out = now > 0x7fffffff ? 0x7fffffff : (int)now;
        }
      }
    }
    __syncthreads();
    const int64_t here0 = before < a.total ? before : a.total;
    before += all;
    pages += took;
    const int64_t here1 = before < a.total ? before : a.total;
    const int64_t t0 = here0 > i0 ? here0 : i0, t1 = here1 < i1 ? here1 : i1;
    for (int64_t i0k = t0 + tid; i0k < t1; i0k += 256 * kTableEach) {
      // the pages of all of the thread's tokens are asked for before any is used
      int64_t t[kTableEach];
      int page[kTableEach], id[kTableEach];
      int32_t* entry[kTableEach];
      bool fresh[kTableEach];
#pragma unroll
      for (int k = 0; k < kTableEach; ++k) {
        const int64_t i = i0k + 256 * k;
        id[k] = -1;
        fresh[k] = false;
        entry[k] = nullptr;
        t[k] = 0;
        if (i >= t1) continue;
        int r = 0;  // the first row whose end lies past i
#pragma unroll
        for (int step = 128; step > 0; step >>= 1)
          if (r_end[r + step - 1] <= i) r += step;
        t[k] = r_len[r] + (i - (r > 0 ? r_end[r - 1] : here0));
        if (t[k] >= cap) continue;
        page[k] = (int)t[k] / a.P;
        entry[k] = a.tables + (int64_t)(b0 + r) * a.t_bs + page[k];
        if (page[k] < r_held[r]) {
          id[k] = *entry[k];
        } else {
          const int64_t at = (int64_t)r_first[r] + page[k] - r_held[r];
          if (at < a.F) id[k] = a.free[at];
          fresh[k] = page[k] * a.P == (int)t[k];  // the page's first token
        }
      }
#pragma unroll
      for (int k = 0; k < kTableEach; ++k) {
        const int64_t i = i0k + 256 * k;
        if (i >= t1) continue;
        if (fresh[k]) *entry[k] = id[k] < 0 ? -1 : id[k];
        int64_t slot = -1;
        if (id[k] >= 0) slot = (int64_t)id[k] * a.P + ((int)t[k] - page[k] * a.P);
        a.slots[i] = slot > 0x7fffffff ? -1 : (int)slot;
        a.positions[i] = t[k] > 0x7fffffff ? 0x7fffffff : (int)t[k];
      }
    }
    if (!last && before >= i1) return;
  }
  // slots behind the last token
  for (int64_t i = (before > i0 ? before : i0) + tid; i < i1; i += 256) {
    a.slots[i] = -1;
    a.positions[i] = 0;
  }
  if (last && tid == 0) {
    a.cu[0] = 0;
    if (state && (before < a.total || a.total == 0)) {
      const int64_t now = taken + (a.total == 0 ? 0 : pages);
      *a.taken_out = now > 0x7fffffff ? 0x7fffffff : (int)now;
    }
  }
}

__global__ __launch_bounds__(256) void k_page_tables(const PageTablesArgs a, int state) {
  const int64_t i0 = (int64_t)blockIdx.x * kTableTokens;
  const int64_t i1 = i0 + kTableTokens < a.total ? i0 + kTableTokens : a.total;
  page_tables(a, i0, i1, blockIdx.x == 0, state);
}
// The new lengths and pages taken alone: where they replace the old ones, which the blocks before read.
__global__ __launch_bounds__(256) void k_page_state(const PageTablesArgs a) { page_tables(a, 0, 0, true, true); }

// ---------------------------------------------------------------------------------------
// The store of new keys and values: 16 bytes of K and of V to a thread. Bound by the bytes, read and written once: the
// stores go past the caches (32771 tokens, 4 heads of 128, [N, HK, P, D] pages, 134 MB: 30.0 -> 21.6 us, 6.2 TB/s; with the
// loads past them too 27.7).
// ---------------------------------------------------------------------------------------

// A block's threads over the 16-byte pieces of a token's heads: `tokens` tokens at once, each thread one piece of one
// (or, where a token has more pieces than threads, every 256th).
struct Pieces {
  int chunks, all, tokens, tok, first;
  __device__ __forceinline__ Pieces(int HK, int D) {
    chunks = D / 8;
    all = HK * chunks;
    tokens = all < 256 ? 256 / all : 1;
    tok = all < 256 ? (int)threadIdx.x / all : 0;
    first = (int)threadIdx.x - tok * all;
  }
  __device__ __forceinline__ bool idle() const { return tok >= tokens; }
};

__global__ __launch_bounds__(256) void k_page_store(const PageStoreArgs a) {
  const Pieces p(a.HK, a.D);
  if (p.idle()) return;
  for (int64_t t = (int64_t)blockIdx.x * p.tokens + p.tok; t < a.T; t += (int64_t)gridDim.x * p.tokens) {
    const int slot = a.slots[t], page = slot / a.P, place = slot - page * a.P;
    if (slot < 0 || page >= a.N) continue;
    for (int c = p.first; c < p.all; c += 256) {
      const int h = c / p.chunks, d = 8 * (c - h * p.chunks);
      u32x4 x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        x[i] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.src[i]) + t * a.s_ts[i] +
                                               h * a.s_hs[i] + d);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        __builtin_nontemporal_store(
            x[i], reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.dst[i].p) + page * a.dst[i].ps +
                                           place * a.dst[i].ts + h * a.dst[i].hs + d));
    }
  }
}

// ---------------------------------------------------------------------------------------
// The beams' states follow their parents, in place: a thread owns 16 bytes of a token of all beams of a request (of
// one layer's K or V), reads what moves from each parent's page and then writes it to the beams' own, so that no
// place is overwritten before it is read, whatever permutation or choice the parents are. Beams that stay are neither
// read nor written, nor are pages that a beam shares with its parent. A block goes through runs of a request's pages, whose
// numbers are read once a run.
//
// Bound by the bytes that move. 12 requests of 8 beams, 358 to 391 tokens, 28 layers, 4 heads of 128, pages of 64 (1.45 GB
// moved): tokens dealt to the threads one at a time, each with its own look at the tables, 472 us; a page to a block and two
// tokens at once 325, four 318, stores past the caches 313; in runs of 16 tokens, whatever the page, 286, an odd
// number of blocks to a request 283 (5.1 TB/s, what a copy reaches). With whole pages, half as many blocks took 358, loads past the caches 370.
//
// A run is 16 tokens, or twice what a block copies at once where that is more. Whole pages / 64 / 32 / 16 tokens: one layer of
// 4 x 8 x 700 tokens in pages of 64 - / 35.7 / 25.4 / 21.3, contiguous caches (a page a row) of 4 beams of 8000 tokens 828 /
// 14.2 / 13.5 / 12.0, 8 x 4 x 4000 801 / 87 / 88 / 84; 4 x 5 x 1800 with 2 heads of 64 - / 17.1 / 17.4 / 21.0.
// ---------------------------------------------------------------------------------------
template <int MOST, int UNROLL>
__global__ __launch_bounds__(256) void k_beam_reorder(const BeamReorderArgs a, int each) {
  const int r = blockIdx.y, layer = blockIdx.z >> 1, cache = blockIdx.z & 1, lane = threadIdx.x & 63;
  const int64_t cap = (int64_t)a.M * a.P;
  const int end = a.lengths[r] < cap ? a.lengths[r] : (int)cap;
  const int start = a.start == nullptr || a.start[r] < 0 ? 0 : a.start[r];
  if (start >= end) return;
  const int runs = (a.P + each - 1) / each;  // of `each` tokens, the last of a page perhaps of fewer
  const int first = start / a.P * runs + start % a.P / each + blockIdx.x;
  const int last = (end - 1) / a.P * runs + (end - 1) % a.P / each;
  if (first > last) return;
  // lane w: the parent of beam w where it moves, else w
  int from = lane;
  if (lane < a.W) {
    const int parent = a.parents[(int64_t)r * a.W + lane];
    if (parent >= 0 && parent < a.W) from = parent;
  }
  if (__ballot(from != lane) == 0) return;
  const Pieces p(a.HK, a.D);
  const int32_t* tables = a.tables + (int64_t)r * a.W * a.t_bs;
  const Pages pg = cache ? a.pages[1] : a.pages[0];
  uint16_t* const pages = static_cast<uint16_t*>(pg.p) + layer * pg.ls;
  for (int run = first; run <= last; run += gridDim.x) {
    const int page = run / runs;
    const int mine = lane < a.W ? tables[(int64_t)lane * a.t_bs + page] : -1;
    const int theirs = __shfl(mine, from);
    const bool moves = theirs != mine && (unsigned)theirs < (unsigned)a.N && (unsigned)mine < (unsigned)a.N;
    const uint64_t go = __ballot(moves);
    if (go == 0) continue;
    // read before the idle threads go on: a wavefront's idle lanes (HK D / 8 = 136 pieces leave 56 in the third) may hold
    // pages of beams, and what the compiler moves or spills behind that branch it moves in the others' lanes only
    int64_t src[MOST], dst[MOST];
#pragma unroll
    for (int w = 0; w < MOST; ++w) {
      src[w] = __builtin_amdgcn_readlane(theirs, w) * pg.ps;
      dst[w] = __builtin_amdgcn_readlane(mine, w) * pg.ps;
    }
    if (p.idle()) continue;
    const int at0 = page * a.P, run0 = (run - page * runs) * each, run1 = run0 + each < a.P ? run0 + each : a.P;
    const int p0 = at0 + run0 > start ? run0 : start - at0;
    const int p1 = run1 < end - at0 ? run1 : end - at0;
    for (int c = p.first; c < p.all; c += 256) {
      const int h = c / p.chunks, d = 8 * (c - h * p.chunks);
      uint16_t* const head = pages + h * pg.hs + d;
      for (int t = p0 + p.tok; t < p1; t += UNROLL * p.tokens) {
        u32x4 v[UNROLL][MOST];
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
          const int tk = t + k * p.tokens;
          uint16_t* const at = head + (tk < p1 ? tk : t) * pg.ts;
#pragma unroll
          for (int w = 0; w < MOST; ++w)
            if (go >> w & 1) v[k][w] = *reinterpret_cast<const u32x4*>(at + src[w]);
        }
#pragma unroll
        for (int k = 0; k < UNROLL; ++k) {
          const int tk = t + k * p.tokens;
          if (tk >= p1) break;
          uint16_t* const at = head + tk * pg.ts;
#pragma unroll
          for (int w = 0; w < MOST; ++w)
            if (go >> w & 1) __builtin_nontemporal_store(v[k][w], reinterpret_cast<u32x4*>(at + dst[w]));
        }
      }
    }
  }
}

}  // namespace

hipError_t launch_page_tables(const PageTablesArgs& a, hipStream_t s) {
  const int64_t blocks = ((int64_t)a.total + kTableTokens - 1) / kTableTokens;
  const bool in_place = a.lengths_out == a.lengths || a.taken_out == a.taken;
  const bool later = in_place && blocks > 1;
  hipLaunchKernelGGL(k_page_tables, dim3((unsigned)(blocks > 0 ? blocks : 1)), dim3(256), 0, s, a, later ? 0 : 1);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !later) return e;
  hipLaunchKernelGGL(k_page_state, dim3(1), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_page_store(const PageStoreArgs& a, hipStream_t s) {
  const int all = a.HK * (a.D / 8), tokens = all < 256 ? 256 / all : 1;
  const int64_t blocks = (a.T + tokens - 1) / tokens;
  hipLaunchKernelGGL(k_page_store, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_beam_reorder(const BeamReorderArgs& a, hipStream_t s) {
  const int all = a.HK * (a.D / 8), at_once = all < 256 ? 256 / all : 1, run = at_once > 8 ? 2 * at_once : 16;
  const int each = a.P < run ? a.P : run;
  // a request's own pages are known on the device only: blocks for 16 of a CU's, up to one to a run of the table's pages
  const int64_t groups = (int64_t)a.R * a.L * 2, most = groups >= 16384 ? 1 : 16384 / groups;
  const int64_t runs = (int64_t)a.M * ((a.P + each - 1) / each);
  // an odd number, so that the requests' first runs, of wide tables all that has work, are not all the same XCDs' (2 x 8
  // beams of 21 tokens in tables of 32 pages, 24 layers, 4 heads of 128: 41.8 -> 15.0 us; 12 x 8 of 390 892 -> 840)
  const dim3 grid((unsigned)(most < runs ? most : runs) | 1u, (unsigned)a.R, (unsigned)(2 * a.L));
  if (a.W <= 4)
    hipLaunchKernelGGL((k_beam_reorder<4, 4>), grid, dim3(256), 0, s, a, each);
  else if (a.W <= 8)
    hipLaunchKernelGGL((k_beam_reorder<8, 4>), grid, dim3(256), 0, s, a, each);
  else if (a.W <= 16)
    hipLaunchKernelGGL((k_beam_reorder<16, 2>), grid, dim3(256), 0, s, a, each);
  else
    hipLaunchKernelGGL((k_beam_reorder<kMostBeams, 1>), grid, dim3(256), 0, s, a, each);
  return hipGetLastError();
}

}  // namespace esep
