// Windowed causal attention with sinks, forward and backward: query i of a sequence sees key j <= i if
// i - j < window or j < sinks. The tile steps, the DMA ring and the layouts are those of the causal
// kernels (attention.hpp, attention_tiles.hpp); what differs is which tiles a block walks, what a
// query sees, and where the blocks run.
//
// Forward and dQ: a block (4 x 32 queries of one kv head, WinItem) of queries q0 .. q1 - 1 walks the tiles of the
// sinks, then those of keys q0 - window + 1 .. q1 - 1 (one run of tiles where the two meet). A wavefront skips
// the 32-key steps that none of its queries sees, and masks only where a border crosses.
//
// dK / dV: a block of 128 keys walks the queries k0 .. k0 + 127 + window - 1. A sink key is also seen by every
// query after that: in a long sequence 32 times as many as another key, which one block would walk
// alone long after the launch's others had ended. Those far queries (i - j >= window) go to blocks of
// their own, kWinFar queries each or more, in the same launch; they and the sink keys' near part write fp32
// partials that k_attn_win_sinks adds in a fixed order. A sequence of up to window + kWinFar tokens has its sink
// keys' blocks walk on to its end instead.
//
// delta = rowsum(dO o) of an o rounded to 16 bits is off by half a step of it, which shows in dQ and dK where a
// query sees few keys (o is then as large as v). The forward can store what o's rounding dropped (o_low), and the
// backward adds it. Errors of dQ and dK in bf16 in the 2-norm against float64: 2.42e-3 instead of 2.57e-3 at a
// window of 16, 2.38e-3 instead of 2.47e-3 at 256 (1.66e-3 is the rounding of the results alone; P and dS, rounded
// to 16 bits for the matrix instructions, make the rest). That costs o_low's bytes: as much memory as o until the
// backward, and 1 to 4% of both passes (forward + backward in us without and with: 65536 tokens, 28 / 4 heads,
// window 1024, bf16 858 + 2990 and 931 + 3053, fp16 898 + 3102 and 964 + 3187; 32768 tokens, 12 / 2 heads, window
// 4096 791 + 2745 and 804 + 2755; 5933 tokens in 8 sequences, window 256 23.0 + 99.4 and 25.6 + 102).
//
// All blocks of a launch do near-equal work, so no order by length is needed: the (sequence, tile,
// head) triples are numbered with the heads innermost and cut into 8 contiguous runs, one to an XCD,
// where neighbouring tiles and the heads of a kv head share K and V in the L2. A sequence's tiles start at a
// number that its offset gives (WinBase), which never overlap and need no sums over the other sequences; the grid
// is sized by T and n_seq whatever max_seqlen is.
//
// Bound by SIMD issue (MFMAs and softmax arithmetic of a wavefront overlap little), and by a block's start where
// its walk is short. In bf16, 12 / 2 heads of 128: 32768 tokens, window 4096, 4 sinks forward 797 us (0.97
// PFLOP/s), backward 2766 (0.70, counting 10 D per pair; S and dP are computed twice, 14 D run); 5933 tokens in 8
// sequences, window 256 25 (0.31) and 104 (0.19).
#include <cmath>
#include <type_traits>

#include "attention_tiles.hpp"

namespace esep {
namespace {

__device__ __forceinline__ int cu_at(const int32_t* cu, int s, int64_t T) {
  const int c = cu[s];
  return c < 0 ? 0 : (c > (int)T ? (int)T : c);
}

// The last sequence s with base(s) <= p, for a base that does not fall, or -1: every lane tests one of 64
// candidates a step, and the wavefront goes on between two of them.
template <class Base>
__device__ __forceinline__ int win_search(int n_seq, int p, Base&& base) {
  const int lane = (int)(threadIdx.x & 63);
  int lo = 0, n = n_seq;
  while (n > 0) {
    const int step = (n + 63) / 64;
    const int64_t at = (int64_t)lane * step;
    const int c = __popcll(__ballot(at < n && base(lo + (int)at) <= p));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    if (step == 1) break;
    n = n - (c - 1) * step < step ? n - (c - 1) * step : step;
  }
  return lo;
}

// The blocks of a sequence that starts at token c are numbered from c * per / 128 + s * pad: per (blocks per
// 128 tokens) and pad such that no sequence has more blocks than numbers.
struct WinBase {
  int per, pad;
  __host__ __device__ __forceinline__ int64_t at(int64_t c, int64_t s) const {
    return ((c * per) >> 7) + s * pad;
  }
};
// 128 keys a block.
constexpr WinBase kWinKeys{1, 1};
// 4 of a sequence's ceil(len / 32) * G items a block: at most G len / 128 + 31 G / 128 + 127 / 128 blocks, and
// two floors are up to 127 / 128 less than G len / 128 apart.
__host__ __device__ __forceinline__ WinBase win_queries(int G) { return {G, (31 * G + 254) / 128}; }

// A block's (sequence, tile, head) among H heads, or a number among the spare blocks.
struct WinPlace {
  int seq, tile, head;   // seq < 0: no work
  int start, end;        // the sequence's tokens
  int rest;              // the first token behind the last sequence
  int spare, n_spare;    // spare >= 0: one of n_spare blocks without a tile (8 or more of them)
};
__device__ __forceinline__ WinPlace win_place(int b, int nblk, int H, const int32_t* cu, int n_seq,
                                              int64_t T, WinBase base) {
  // the offsets of up to 63 sequences in one read, a lane each: a block's place then costs one trip to memory
  const int lane = (int)(threadIdx.x & 63);
  const bool few = n_seq < 64;
  const int mine = few ? cu_at(cu, lane < n_seq ? lane : n_seq, T) : 0;
  const int rest = few ? __builtin_amdgcn_readlane(mine, n_seq) : cu_at(cu, n_seq, T);
  const int live = (int)base.at(rest, n_seq) * H;
  const int per = (live + 7) / 8, xcd = b & 7, slot = b >> 3;
  WinPlace w{-1, 0, 0, 0, 0, rest, -1, nblk - 8 * per};
  if (slot >= per) {
    w.spare = 8 * (slot - per) + xcd;
    return w;
  }
  const int i = xcd * per + slot;
  if (i >= live) return w;
  const int p = i / H;
  int s;
  if (few) {
    s = __popcll(__ballot(lane < n_seq && base.at(mine, lane) <= p)) - 1;
    if (s < 0) return w;
    w.start = __builtin_amdgcn_readlane(mine, s);
    w.end = __builtin_amdgcn_readlane(mine, s + 1);
  } else {
    s = win_search(n_seq, p, [&](int j) { return base.at(cu_at(cu, j, T), j); });
    if (s < 0) return w;
    w.start = cu_at(cu, s, T);
    w.end = cu_at(cu, s + 1, T);
  }
  if (w.end < w.start) w.end = w.start;
  w.seq = s;
  w.tile = p - (int)base.at(w.start, s);
  w.head = i - p * H;
  return w;
}
inline int64_t win_blocks(int64_t T, int n_seq, int64_t H, WinBase base) {
  return (base.at(T, n_seq) * H + 7) / 8 * 8 + 8;
}

// out = 0 for the tokens behind the last sequence (W elements each, W a multiple of 8), dealt to the
// spare blocks.
template <typename T>
__device__ __forceinline__ void zero_rest(T* out, int64_t rs, int W, int from, int64_t rows,
                                          const WinPlace& w) {
  const int chunks = W / 8;
  const int64_t n = (rows - from) * chunks;
  for (int64_t i = (int64_t)w.spare * kAttnThreads + threadIdx.x; i < n;
       i += (int64_t)w.n_spare * kAttnThreads) {
    const int64_t t = from + i / chunks;
    *reinterpret_cast<uint4*>(out + t * rs + 8 * (i % chunks)) = make_uint4(0, 0, 0, 0);
  }
}

// A wavefront's 32 queries of one head. A block's 4 wavefronts take 4 of a kv head's (32 queries, head) items,
// the heads innermost: with 3 and more query heads to a kv head a block spans at most 64 queries, and walks
// window + 64 keys where 128 queries of one head walk window + 128 (of which a wavefront sees window + 32). 32768
// tokens in 4 sequences, 28 / 4 heads, window 128, bf16: forward 171 us against 200, backward 614 against 708;
// 65536 tokens at window 1024 869 against 912 and 3047 against 3104.
struct WinItem {
  int q0, q1;   // the block's queries
  int qw0, h;   // the wavefront's first query (past the end: none) and head
  __device__ __forceinline__ WinItem(const WinPlace& pl, int G, int w) {
    const int n = (pl.end - pl.start + 31) / 32;
    const int s0 = 4 * pl.tile / G, s1 = (4 * pl.tile + 3) / G, i = 4 * pl.tile + w, s = i / G;
    q0 = s0 < n ? pl.start + 32 * s0 : pl.end;
    q1 = s1 + 1 < n ? pl.start + 32 * (s1 + 1) : pl.end;
    qw0 = s < n ? pl.start + 32 * s : pl.end;
    h = pl.head * G + i - s * G;
  }
};

// The key tiles of a block of queries q0 .. q1 - 1: `ns` tiles of the sinks from `start`, then tiles from `lo` to
// kend. Where the sinks reach the window they are one run.
struct KeyWalk {
  int start, lo, kend, sink_hi, ns, n;
  template <int BN>
  __device__ __forceinline__ void init(int start_, int end, int q0, int q1, int window, int sinks) {
    start = start_;
    sink_hi = start + (sinks < end - start ? sinks : end - start);
    kend = q1;
    lo = q0 - window + 1;
    if (lo <= sink_hi) lo = start;
    ns = lo > start ? (sink_hi - start + BN - 1) / BN : 0;
    n = ns + (kend - lo + BN - 1) / BN;
  }
};

// Walks the tiles of a block: K and V through a ring of two LDS buffers (tile t + 1 in flight while
// tile t is consumed), step(ks, vs, kh, utop, top) for every 32 keys that the wavefront sees.
template <typename T, int D, int BN, class Step>
__device__ __forceinline__ void walk_keys(const AttnArgs& a, const KeyWalk& kw, int kvh, int window,
                                          char (&kv)[2][2][BN * 2 * D], int lane, int w, int qw0,
                                          int qi, int end, Step&& step) {
  constexpr int RB = 2 * D;
  const bool wave_live = qw0 < end;
  const int wq_last = qw0 + 31 < end ? qw0 + 31 : end - 1;
  const char* kbase = reinterpret_cast<const char*>(static_cast<const T*>(a.k) + (int64_t)kvh * D);
  const char* vbase = reinterpret_cast<const char*>(static_cast<const T*>(a.v) + (int64_t)kvh * D);
  SwzFill<BN, 4, RB> fk(lane, w, a.k_rs * (int64_t)sizeof(T)), fv(lane, w, a.v_rs * (int64_t)sizeof(T));
  fk.seq_begin(kbase, kw.lo);
  fv.seq_begin(vbase, kw.lo);
  auto issue = [&](int buf, int t) {
    const int kt = t < kw.ns ? kw.start + t * BN : kw.lo + (t - kw.ns) * BN;
    const int rend = t < kw.ns ? kw.sink_hi : kw.kend;
    if (t >= kw.ns && kt + BN <= rend) {
      fk.seq_whole(kv[buf][0]);
      fv.seq_whole(kv[buf][1]);
    } else {
      swz_fill2(fk, kv[buf][0], kbase, fv, kv[buf][1], vbase, kt, rend);
    }
  };
  if (kw.n > 0) issue(0, 0);
  auto tile = [&](int t, auto bc) {
    constexpr int B = decltype(bc)::value;
    // this wavefront's DMA of tile t has landed; the barrier publishes every wavefront's rows
    // and certifies that tile t - 1, in the other buffer, is consumed
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    __syncthreads();
    if (t + 1 < kw.n) issue(B ^ 1, t + 1);
    const bool sink = t < kw.ns;
    const int kt = sink ? kw.start + t * BN : kw.lo + (t - kw.ns) * BN;
    const int utop = sink ? kw.sink_hi - 1 : qw0, top = sink ? kw.sink_hi - 1 : qi;
    const int last = sink ? kw.sink_hi - 1 : wq_last;
#pragma unroll
    for (int h = 0; h < BN / 32; ++h) {
      const int kh = kt + 32 * h;
      if (!wave_live || kh > last) return;
      if (kh + 31 <= qw0 - window && kh >= kw.sink_hi) continue;
      step(kv[B][0] + 32 * RB * h, kv[B][1] + 32 * RB * h, kh, utop, top);
    }
  };
  int t = 0;
  for (; t + 1 < kw.n; t += 2) {
    tile(t, std::integral_constant<int, 0>{});
    tile(t + 1, std::integral_constant<int, 1>{});
  }
  if (t < kw.n) tile(t, std::integral_constant<int, 0>{});
}

template <typename T, int D, int BN>
__global__ __launch_bounds__(kAttnThreads, kFwdPerCU<D>) void k_attn_win_fwd(const AttnWinArgs p) {
  using V8 = typename Mfma<T>::v8;
  const AttnArgs& a = p.b.f;
  __shared__ __align__(1024) char kv[2][2][BN * 2 * D];  // [buffer][K, V][swizzled rows]

  const WinPlace pl = win_place(attn_block(), (int)(gridDim.x * gridDim.y), a.HK, a.cu, a.n_seq, a.T,
                                win_queries(a.HQ / a.HK));
  if (pl.spare >= 0 && p.zero_rest)
    zero_rest<T>(static_cast<T*>(a.o), a.o_rs, a.HQ * D, pl.rest, a.T, pl);
  if (pl.seq < 0) return;
  const int start = pl.start, end = pl.end;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const WinItem it(pl, a.HQ / a.HK, w);
  if (it.q0 >= end) return;
  const int lq = lane & 31, hi = lane >> 5;
  const int h = it.h, qw0 = it.qw0, qi = qw0 + lq;

  V8 qb[D / 16];
  {
    const T* qrow = static_cast<const T*>(a.q) + (int64_t)qi * a.q_rs + (int64_t)h * D + 8 * hi;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      qb[c] = qi < end ? ld16<V8>(qrow + 16 * c) : V8{};
  }
  f32x16 oacc[D / 32];
#pragma unroll
  for (int md = 0; md < D / 32; ++md) oacc[md] = f32x16{};
  float m = -INFINITY, l = 0.f;
  KeyWalk kw;
  kw.init<BN>(start, end, it.q0, it.q1, p.window, p.sinks);
  walk_keys<T, D, BN>(a, kw, pl.head, p.window, kv, lane, w, qw0, qi, end,
                      [&](const char* ks, const char* vs, int kh, int utop, int top)
                          __attribute__((always_inline)) {
                        fwd_tile_swz<T, D>(ks, vs, lane, a.scale_log2, qb, oacc, m, l,
                                           [&](f32x16& acc) __attribute__((always_inline)) {
                                             mask_window(acc, kh, utop, qw0 + 31 - p.window, top,
                                                         qi - p.window, kw.sink_hi, hi);
                                           });
                      });
  if (qi >= end) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  store_rows_t<T, D>(static_cast<T*>(a.o) + (int64_t)qi * a.o_rs + (int64_t)h * D, oacc, hi, inv);
  if (a.o_low != nullptr)
    store_low_t<T, D>(static_cast<T*>(a.o_low) + ((int64_t)qi * a.HQ + h) * D, oacc, hi, inv);
  if (hi == 0 && a.lse != nullptr)
    a.lse[(int64_t)h * a.T + qi] = (m + log2f(l)) * 0.69314718055994531f;
}

template <typename T, int D, int BN>
__global__ __launch_bounds__(kAttnThreads, kDqPerCU<D>) void k_attn_win_dq(const AttnWinArgs p) {
  using V8 = typename Mfma<T>::v8;
  const AttnBwdArgs& b = p.b;
  const AttnArgs& a = b.f;
  __shared__ __align__(1024) char kv[2][2][BN * 2 * D];

  const WinPlace pl = win_place(attn_block(), (int)(gridDim.x * gridDim.y), a.HK, a.cu, a.n_seq, a.T,
                                win_queries(a.HQ / a.HK));
  if (pl.spare >= 0)
    zero_rest<T>(static_cast<T*>(b.dq), b.dq_rs, a.HQ * D, pl.rest, a.T, pl);
  if (pl.seq < 0) return;
  const int start = pl.start, end = pl.end;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const WinItem it(pl, a.HQ / a.HK, w);
  if (it.q0 >= end) return;
  const int lq = lane & 31, hi = lane >> 5;
  const int h = it.h, qw0 = it.qw0, qi = qw0 + lq;
  const bool qok = qi < end;

  V8 qb[D / 16], db[D / 16];
  float delta = 0.f;
  {
    const int64_t col = (int64_t)h * D + 8 * hi;
    const T* qrow = static_cast<const T*>(a.q) + (int64_t)qi * a.q_rs + col;
    const T* drow = static_cast<const T*>(b.dout) + (int64_t)qi * b.do_rs + col;
    const T* orow = static_cast<const T*>(a.o) + (int64_t)qi * a.o_rs + col;
    const bool low = a.o_low != nullptr;
    const T* lrow = static_cast<const T*>(a.o_low) + (int64_t)qi * a.HQ * D + col;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      qb[c] = qok ? ld16<V8>(qrow + 16 * c) : V8{};
      db[c] = qok ? ld16<V8>(drow + 16 * c) : V8{};
      const V8 o8 = qok ? ld16<V8>(orow + 16 * c) : V8{};
      const V8 l8 = low && qok ? ld16<V8>(lrow + 16 * c) : V8{};
#pragma unroll
      for (int e = 0; e < 8; ++e)
        delta = fmaf((float)db[c][e], (float)o8[e] + (float)l8[e], delta);
    }
    delta = pair_sum(delta);
    if (qok && hi == 0) b.delta[(int64_t)h * a.T + qi] = delta;
  }
  const float lse2 = qok ? a.lse[(int64_t)h * a.T + qi] * kLog2e : 0.f;
  f32x16 dqa[D / 32];
#pragma unroll
  for (int md = 0; md < D / 32; ++md) dqa[md] = f32x16{};
  KeyWalk kw;
  kw.init<BN>(start, end, it.q0, it.q1, p.window, p.sinks);
  walk_keys<T, D, BN>(a, kw, pl.head, p.window, kv, lane, w, qw0, qi, end,
                      [&](const char* ks, const char* vs, int kh, int utop, int top)
                          __attribute__((always_inline)) {
                        dq_tile_swz<T, D>(ks, vs, lane, a.scale_log2, lse2, delta, qb, db, dqa,
                                          [&](f32x16& s) __attribute__((always_inline)) {
                                            mask_window(s, kh, utop, qw0 + 31 - p.window, top,
                                                        qi - p.window, kw.sink_hi, hi);
                                          });
                      });
  if (!qok) return;
  store_rows_t<T, D>(static_cast<T*>(b.dq) + (int64_t)qi * b.dq_rs + (int64_t)h * D, dqa, hi,
                     a.scale);
}

// 32 queries of the dK / dV walk for a wavefront's 32 keys: the query rows at qrow / drow (Q and dO,
// 32 rows of the swizzled LDS tiles), their lse and delta words, the keys' K operands in registers and
// their V rows at vlds. s[i] is S[q][key] for query row 8 (i / 4) + 4 hi + i % 4; mask(s) sets what the
// lane's key is not seen by to -inf. rop is the lane's row operand offset (swz_row_base). P and dS are rounded to
// T, the matrix instructions' operand type.
template <typename T, int D, class Mask>
__device__ __forceinline__ void dkdv_tile_swz(const char* qrow, const char* drow, const char* vlds,
                                              const float* lse_s, const float* del_s, int hi,
                                              float scale_log2, uint32_t rop,
                                              const SwzTr<2 * D>& trd,
                                              const typename Mfma<T>::v8 (&kb)[D / 16],
                                              f32x16 (&dka)[D / 32], f32x16 (&dva)[D / 32],
                                              Mask&& mask) {
  using V8 = typename Mfma<T>::v8;
  auto rowc = [&](int c) __attribute__((always_inline)) -> uint32_t { return rop ^ (32u * c); };
  __builtin_amdgcn_s_setprio(1);  // MFMA runs at raised priority, as in the forward
  f32x16 s = f32x16{}, dp = f32x16{};
  {
    // operands read two chunks ahead, pinned by scheduling barriers (the largest read-ahead
    // that fits 256 registers: config 5 backward 5.02 -> 4.95 ms)
    constexpr int RA = 2;
    V8 qbf[RA], dbf[RA], vbf[RA];
#pragma unroll
    for (int c = 0; c < RA; ++c) {
      qbf[c] = ld16<V8>(qrow + rowc(c));
      dbf[c] = ld16<V8>(drow + rowc(c));
      vbf[c] = ld16<V8>(vlds + rowc(c));
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      s = Mfma<T>::run(qbf[c % RA], kb[c], s);
      dp = Mfma<T>::run(dbf[c % RA], vbf[c % RA], dp);
      if (c + RA < D / 16) {
        qbf[c % RA] = ld16<V8>(qrow + rowc(c + RA));
        dbf[c % RA] = ld16<V8>(drow + rowc(c + RA));
        vbf[c % RA] = ld16<V8>(vlds + rowc(c + RA));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __builtin_amdgcn_s_setprio(0);
  mask(s);
  V8 pb[2], sb_[2];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 l4 = *reinterpret_cast<const float4*>(&lse_s[8 * j + 4 * hi]);
    const float4 d4 = *reinterpret_cast<const float4*>(&del_s[8 * j + 4 * hi]);
    const float lr[4] = {l4.x, l4.y, l4.z, l4.w}, dr[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = 4 * j + e;
      const float p = exp2_fast(fmaf(s[i], scale_log2, -lr[e] * kLog2e));
      pb[i / 8][i % 8] = (T)p;
      sb_[i / 8][i % 8] = (T)(p * (dp[i] - dr[e]));
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_setprio(1);
  // dV^T += dO^T P and dK^T += Q^T dS, queries in the permuted order of pb / sb_: operand
  // pair i = (md, c2) = (i / 2, i % 2) read RB pairs ahead, pinned by scheduling barriers
  // (the compiler kept one pair ahead: config-5-like backward 4.66 -> 4.56 ms, the same
  // bits; three ahead, or the first pairs read before the exponentials, spill at 256
  // registers)
  constexpr int RB = 2;
  V8 dotb[RB], qtb[RB];
  auto rd = [&](int i, int slot) {
    const int md = i >> 1, rb = 16 * (i & 1);
    dotb[slot] = trd.template read<V8>(drow, rb, md);
    qtb[slot] = trd.template read<V8>(qrow, rb, md);
  };
#pragma unroll
  for (int i = 0; i < RB; ++i) rd(i, i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < 2 * (D / 32); ++i) {
    const int md = i >> 1, c2 = i & 1;
    dva[md] = Mfma<T>::run(dotb[i % RB], pb[c2], dva[md]);
    dka[md] = Mfma<T>::run(qtb[i % RB], sb_[c2], dka[md]);
    if (i + RB < 2 * (D / 32)) rd(i + RB, i % RB);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

// The places of a sequence's sink partials (attention.hpp: WinSlots); it starts at token c.
__device__ __forceinline__ int win_main_base(const AttnWinArgs& p, int seq, int c) {
  return p.by_seq ? seq : (int)(c / ((int64_t)p.window + kWinFar));
}
__device__ __forceinline__ int win_far_base(const AttnWinArgs& p, int seq, int c) {
  return c / p.far_len + win_main_base(p, seq, c);
}

// fp32 dK^T / scale and dV^T of a lane's key into partial `idx` of a sink buffer, [idx][HK][2][sinks][D].
template <int D>
__device__ __forceinline__ void store_sink(float* buf, int64_t idx, int HK, int kh, int sinks, int r,
                                           int hi, const f32x16 (&dka)[D / 32],
                                           const f32x16 (&dva)[D / 32]) {
  float* pk = buf + (((idx * HK + kh) * 2) * sinks + r) * D + 4 * hi;
  float* pv = pk + (int64_t)sinks * D;
#pragma unroll
  for (int md = 0; md < D / 32; ++md)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *reinterpret_cast<float4*>(pk + 32 * md + 8 * j) =
          make_float4(dka[md][4 * j], dka[md][4 * j + 1], dka[md][4 * j + 2], dka[md][4 * j + 3]);
      *reinterpret_cast<float4*>(pv + 32 * md + 8 * j) =
          make_float4(dva[md][4 * j], dva[md][4 * j + 1], dva[md][4 * j + 2], dva[md][4 * j + 3]);
    }
}

template <typename T, int D>
__global__ __launch_bounds__(kAttnThreads, D == 128 ? kDkdvPerCU : 3) void k_attn_win_dkdv(const AttnWinArgs p) {
  constexpr int NW = 4, BQ = 32, BK = kAttnBM, ROWB = 2 * D;
  using V8 = typename Mfma<T>::v8;
  const AttnBwdArgs& b = p.b;
  const AttnArgs& a = b.f;
  __shared__ __align__(1024) char qs[2][BQ * ROWB];
  __shared__ __align__(1024) char ds_[2][BQ * ROWB];
  __shared__ __align__(16) float ld_s[2][2 * BQ];  // lse, then delta
  __shared__ __align__(1024) char vsm[BK * ROWB];

  const int G = a.HQ / a.HK, bid = attn_block();
  const bool far = bid >= p.n_main;
  if (far && !p.far) return;
  int seq, kh, part, parts, tile, chunk = 0, start = 0, end = 0;
  if (!far) {
    const WinPlace pl = win_place(bid, p.n_main, a.HK * b.split, a.cu, a.n_seq, a.T, kWinKeys);
    if (pl.spare >= 0) {
      zero_rest<T>(static_cast<T*>(b.dk), b.dk_rs, a.HK * D, pl.rest, a.T, pl);
      zero_rest<T>(static_cast<T*>(b.dv), b.dv_rs, a.HK * D, pl.rest, a.T, pl);
    }
    seq = pl.seq;
    start = pl.start;
    end = pl.end;
    kh = pl.head / b.split;
    part = pl.head % b.split;
    tile = pl.tile;
    parts = b.split;
  } else {
    const int kts = (p.sinks + BK - 1) / BK, per = kts * a.HK * p.far_split;
    const int slot = (bid - p.n_main) / per, r = (bid - p.n_main) % per;
    seq = win_search(a.n_seq, slot,
                     [&](int j) { return win_far_base(p, j, cu_at(a.cu, j, a.T)); });
    if (seq >= 0) {
      seq_bounds(a.cu, seq, a.T, &start, &end);
      chunk = slot - win_far_base(p, seq, start);
    }
    tile = r % kts;
    kh = r / kts % a.HK;
    part = r / kts / a.HK;
    parts = p.far_split;
  }
  if (seq < 0) return;
  const int len = end - start;
  const bool lng = p.far && len - kWinFar > p.window;  // its sink keys have far blocks
  const int sink_hi = start + (p.sinks < len ? p.sinks : len);
  const int k0 = start + tile * BK;
  const int kend = far ? sink_hi : end;  // this block's keys end here
  if (k0 >= kend) return;
  // the block's queries [qa, qe)
  int qa = k0, qe = end;
  if (far) {
    if (!lng || (int64_t)chunk * p.far_len >= len - p.window) return;
    qa = start + p.window + chunk * p.far_len;
    qe = end - qa < p.far_len ? end : qa + p.far_len;
    if (qe <= k0 + p.window) return;
  } else if ((lng || k0 >= sink_hi) && end - k0 - (BK - 1) > p.window) {
    qe = k0 + BK - 1 + p.window;
  }
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int lq = lane & 31, hi = lane >> 5;
  const int kw0 = k0 + 32 * w, kj = kw0 + lq;
  const bool kok = kj < kend, wave_live = kw0 < kend;
  const int g0 = part * G / parts, gs = (part + 1) * G / parts - g0, h0 = kh * G + g0;
  // the queries that see this lane's key in this block: tlo <= t < thi; wlo, wmin and wmax are the
  // wavefront's greatest tlo and least and greatest thi
  const bool open = !lng || far;  // a sink key is seen to the end
  auto last_of = [&](int k) { return (open && k < sink_hi) || qe - k < p.window ? qe : k + p.window; };
  const int tlo = far ? kj + p.window : kj, thi = last_of(kj);
  const int wlo0 = far ? kw0 + p.window : kw0, wlo = wlo0 + 31;
  const int wfirst = last_of(kw0), wlast = last_of(kw0 + 31);
  const int wmin = open && kw0 < sink_hi && kw0 + 31 >= sink_hi ? last_of(sink_hi)
                                                                : wfirst;
  const int wmax = wfirst > wlast ? wfirst : wlast;

  V8 kb[D / 16];
  {
    const T* krow = static_cast<const T*>(a.k) + (int64_t)kj * a.k_rs + (int64_t)kh * D + 8 * hi;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) kb[c] = kok ? ld16<V8>(krow + 16 * c) : V8{};
  }
  {
    TileRows<T, D, BK, kAttnThreads> vr;
    vr.load(static_cast<const T*>(a.v) + (int64_t)kh * D, a.v_rs, k0, kend, tid);
    vr.store_swz(vsm, tid);
  }
  const uint32_t rop = swz_row_base<ROWB>(lane);
  const char* vlds = vsm + 32 * w * ROWB;
  const SwzTr<ROWB> trd(lane);
  f32x16 dka[D / 32], dva[D / 32];
#pragma unroll
  for (int md = 0; md < D / 32; ++md) dka[md] = dva[md] = f32x16{};

  const int nqt = (qe - qa + BQ - 1) / BQ, items = gs * nqt;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  SwzFill<BQ, NW, ROWB> fq(lane, wu, a.q_rs * (int64_t)sizeof(T));
  SwzFill<BQ, NW, ROWB> fd(lane, wu, b.do_rs * (int64_t)sizeof(T));
  auto issue = [&](int it, int buf) {
    const int h = h0 + it / nqt, qt = qa + (it % nqt) * BQ;
    const int64_t col = (int64_t)h * D;
    const char* qbase = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + col);
    const char* dbase = reinterpret_cast<const char*>(static_cast<const T*>(b.dout) + col);
    if (it % nqt == 0) {
      fq.seq_begin(qbase, qa);
      fd.seq_begin(dbase, qa);
    }
    if (qt + BQ <= end) {
      fq.seq_whole(qs[buf]);
      fd.seq_whole(ds_[buf]);
    } else {
      swz_fill2(fq, qs[buf], qbase, fd, ds_[buf], dbase, qt, end);
    }
    if (wu == 0) {
      const int t0 = qt + (lane & 31);  // word `lane` of [lse | delta]
      const int t = t0 < end ? t0 : end - 1;
      lds_dma_dword((lane < 32 ? a.lse : b.delta) + (int64_t)h * a.T + t, &ld_s[buf][0]);
    }
  };
  if (items > 0) issue(0, 0);
  for (int it = 0; it < items; ++it) {
    const int qt = qa + (it % nqt) * BQ, buf = it & 1;
    __builtin_amdgcn_s_waitcnt(kWaitVm0);
    __syncthreads();
    if (it + 1 < items) issue(it + 1, buf ^ 1);
    if (!wave_live || qt + BQ - 1 < wlo0 || qt >= wmax) continue;
    dkdv_tile_swz<T, D>(qs[buf], ds_[buf], vlds, ld_s[buf], ld_s[buf] + BQ, hi, a.scale_log2, rop, trd,
                        kb, dka, dva, [&](f32x16& s) __attribute__((always_inline)) {
                          if (qt < wlo || qt + 31 >= wmin) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                              const int t = qt + 8 * (i / 4) + 4 * hi + (i % 4);
                              if (t < tlo || t >= thi) s[i] = -INFINITY;
                            }
                          }
                        });
  }
  if (!kok) return;
  if (far) {
    const int64_t idx = (int64_t)(win_far_base(p, seq, start) + chunk) * p.far_split + part;
    store_sink<D>(p.sink_far, idx, a.HK, kh, p.sinks, kj - start, hi, dka, dva);
    return;
  }
  if (lng && kj < sink_hi) {
    const int64_t idx = (int64_t)win_main_base(p, seq, start) * b.split + part;
    store_sink<D>(p.sink_main, idx, a.HK, kh, p.sinks, kj - start, hi, dka, dva);
    return;
  }
  if (b.split == 1) {
    store_rows_t<T, D>(static_cast<T*>(b.dk) + (int64_t)kj * b.dk_rs + (int64_t)kh * D, dka, hi,
                       a.scale);
    store_rows_t<T, D>(static_cast<T*>(b.dv) + (int64_t)kj * b.dv_rs + (int64_t)kh * D, dva, hi,
                       1.f);
    return;
  }
  // fp32 partials [2][split][T][HK][D], as the causal kernel's
  const int64_t plane = a.T * a.HK * D;
  float* pk = b.part + (int64_t)part * plane + ((int64_t)kj * a.HK + kh) * D + 4 * hi;
  float* pv = pk + (int64_t)b.split * plane;
#pragma unroll
  for (int md = 0; md < D / 32; ++md)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      *reinterpret_cast<float4*>(pk + 32 * md + 8 * j) =
          make_float4(dka[md][4 * j], dka[md][4 * j + 1], dka[md][4 * j + 2], dka[md][4 * j + 3]);
      *reinterpret_cast<float4*>(pv + 32 * md + 8 * j) =
          make_float4(dva[md][4 * j], dva[md][4 * j + 1], dva[md][4 * j + 2], dva[md][4 * j + 3]);
    }
}

// dK = scale * sum dK_s, dV = sum dV_s over the split partials, s ascending, for every token of a
// sequence; 0 behind the last. (Sink rows that have partials of their own follow.)
template <typename T>
__global__ __launch_bounds__(256) void k_attn_win_reduce(const AttnWinArgs p, int D) {
  const AttnBwdArgs& b = p.b;
  const int64_t row = (int64_t)b.f.HK * D, plane = b.f.T * row;
  const int64_t e = 4 * ((int64_t)blockIdx.x * blockDim.x + threadIdx.x);
  if (e >= plane) return;
  const int64_t t = e / row, r = e % row;
  const bool live = t < cu_at(b.f.cu, b.f.n_seq, b.f.T);
  for (int which = 0; which < 2; ++which) {
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live) {
      const float* src = b.part + (int64_t)which * b.split * plane + e;
      acc = *reinterpret_cast<const float4*>(src);
      for (int s = 1; s < b.split; ++s) {
        const float4 v = *reinterpret_cast<const float4*>(src + (int64_t)s * plane);
        acc.x += v.x;
        acc.y += v.y;
        acc.z += v.z;
        acc.w += v.w;
      }
    }
    const float mul = which == 0 ? b.f.scale : 1.f;
    T o4[4] = {(T)(acc.x * mul), (T)(acc.y * mul), (T)(acc.z * mul), (T)(acc.w * mul)};
    T* dst = static_cast<T*>(which == 0 ? b.dk : b.dv) + t * (which == 0 ? b.dk_rs : b.dv_rs) + r;
    *reinterpret_cast<uint2*>(dst) = __builtin_bit_cast(uint2, o4);
  }
}

// The sink rows of the long sequences: near partials, then the far ones by chunk and part. One block per
// (sequence, kv head, dK or dV, row); D / 4 lanes across, the partials dealt to the block's groups,
// whose sums are added in their order.
template <typename T, int D>
__global__ __launch_bounds__(256) void k_attn_win_sinks(const AttnWinArgs p) {
  constexpr int QUADS = D / 4, GROUPS = 256 / QUADS;
  __shared__ float4 sums[GROUPS][QUADS];
  const AttnBwdArgs& b = p.b;
  const AttnArgs& a = b.f;
  const int r = (int)(blockIdx.x % p.sinks), which = (int)(blockIdx.x / p.sinks % 2);
  const int kh = (int)(blockIdx.x / p.sinks / 2 % a.HK), slot = (int)(blockIdx.x / p.sinks / 2 / a.HK);
  const int seq = win_search(a.n_seq, slot,
                             [&](int j) { return win_main_base(p, j, cu_at(a.cu, j, a.T)); });
  if (seq < 0) return;
  int start, end;
  seq_bounds(a.cu, seq, a.T, &start, &end);
  const int len = end - start;
  if (len - kWinFar <= p.window || r >= len || win_main_base(p, seq, start) != slot) return;
  // chunks whose far block wrote this row: those with a query that sees a key of its tile from afar
  const int off = r / kAttnBM * kAttnBM;
  const int first = off / p.far_len, chunks = (int)(((int64_t)len - p.window + p.far_len - 1) / p.far_len);
  const int n = b.split + (len - p.window > off ? (chunks - first) * p.far_split : 0);
  const int64_t stride = (int64_t)a.HK * 2 * p.sinks * D;
  const int g = threadIdx.x / QUADS, x = threadIdx.x % QUADS;
  const int64_t at = ((int64_t)(kh * 2 + which) * p.sinks + r) * D + 4 * x;
  const float* near = p.sink_main + (int64_t)slot * b.split * stride + at;
  const float* away = p.sink_far +
                      (int64_t)(win_far_base(p, seq, start) + first) * p.far_split * stride + at;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = g; i < n; i += GROUPS) {
    const float* src = i < b.split ? near + i * stride : away + (i - b.split) * stride;
    const float4 v = *reinterpret_cast<const float4*>(src);
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  sums[g][x] = acc;
  __syncthreads();
  if (g != 0) return;
  for (int i = 1; i < GROUPS; ++i) {
    const float4 v = sums[i][x];
    acc.x += v.x;
    acc.y += v.y;
    acc.z += v.z;
    acc.w += v.w;
  }
  const float mul = which == 0 ? a.scale : 1.f;
  T o4[4] = {(T)(acc.x * mul), (T)(acc.y * mul), (T)(acc.z * mul), (T)(acc.w * mul)};
  T* dst = static_cast<T*>(which == 0 ? b.dk : b.dv) +
           (int64_t)(start + r) * (which == 0 ? b.dk_rs : b.dv_rs) + (int64_t)kh * D + 4 * x;
  *reinterpret_cast<uint2*>(dst) = __builtin_bit_cast(uint2, o4);
}

__global__ __launch_bounds__(256) void k_attn_rest(const AttnRestArgs a) {
  const int from = cu_at(a.cu, a.n_seq, a.T), i = blockIdx.y;
  if (a.t[i] == nullptr) return;
  const int chunks = a.w[i] / 8;  // of 16 bytes
  const int64_t n = (a.T - from) * chunks;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n;
       e += (int64_t)gridDim.x * blockDim.x)
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.t[i]) + (from + e / chunks) * a.rs[i] +
                              8 * (e % chunks)) = make_uint4(0, 0, 0, 0);
}

// Blocks of 256 threads that a one-dimensional grid takes (it counts its threads in 32 bits).
constexpr int64_t kWinMaxSums = (int64_t{1} << 24) - 1;

template <typename T, int D>
hipError_t fwd_run(const AttnWinArgs& p, hipStream_t s) {
  const AttnArgs& f = p.b.f;
  const int64_t n = win_blocks(f.T, f.n_seq, f.HK, win_queries(f.HQ / f.HK));
  if (!attn_grid_ok(n)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((k_attn_win_fwd<T, D, D == 128 ? 32 : 64>), attn_grid(n), dim3(kAttnThreads), 0, s,
                     p);
  return hipGetLastError();
}

struct WinGrids {
  int64_t nq, nk, nfar, nsum;
  explicit WinGrids(const AttnWinArgs& p) {
    const AttnArgs& f = p.b.f;
    const int64_t tiles = ((int64_t)p.sinks + kAttnBM - 1) / kAttnBM;
    const WinSlots w = win_slots(f.T, f.n_seq, f.HK, p.window, p.sinks);
    nq = win_blocks(f.T, f.n_seq, f.HK, win_queries(f.HQ / f.HK));
    nk = win_blocks(f.T, f.n_seq, (int64_t)f.HK * p.b.split, kWinKeys);
    nfar = p.far ? w.far * tiles * f.HK * p.far_split : 0;
    nsum = p.far ? w.main * f.HK * 2 * p.sinks : 0;
  }
  bool ok() const { return attn_grid_ok(nq) && attn_grid_ok(nk + nfar) && nsum <= kWinMaxSums; }
};

template <typename T, int D>
hipError_t bwd_run(const AttnWinArgs& a, hipStream_t s) {
  AttnWinArgs p = a;
  const AttnArgs& f = p.b.f;
  const WinGrids g(p);
  if (!g.ok()) return hipErrorInvalidValue;
  const int64_t nq = g.nq, nk = g.nk, nfar = g.nfar, nsum = g.nsum;
  p.n_main = (int)nk;
  hipLaunchKernelGGL((k_attn_win_dq<T, D, D == 128 ? 32 : 64>), attn_grid(nq), dim3(kAttnThreads), 0, s,
                     p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((k_attn_win_dkdv<T, D>), attn_grid(nk + nfar), dim3(kAttnThreads), 0, s, p);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.b.split > 1) {
    const int64_t quads = f.T * f.HK * D / 4;
    hipLaunchKernelGGL((k_attn_win_reduce<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, p,
                       D);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.far) {
    hipLaunchKernelGGL((k_attn_win_sinks<T, D>), dim3((unsigned)nsum), dim3(256), 0, s, p);
    e = hipGetLastError();
  }
  return e;
}

template <typename T>
hipError_t fwd_d(const AttnWinArgs& a, int D, hipStream_t s, bool* sup) {
  *sup = D == 128 || D == 64;
  if (D == 128) return fwd_run<T, 128>(a, s);
  if (D == 64) return fwd_run<T, 64>(a, s);
  return hipErrorInvalidValue;
}
template <typename T>
hipError_t bwd_d(const AttnWinArgs& a, int D, hipStream_t s, bool* sup) {
  *sup = D == 128 || D == 64;
  if (D == 128) return bwd_run<T, 128>(a, s);
  if (D == 64) return bwd_run<T, 64>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_attn_rest(const AttnRestArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(k_attn_rest, dim3(64, 3), dim3(256), 0, s, a);
  return hipGetLastError();
}

bool attn_win_bwd_fits(const AttnWinArgs& p) { return WinGrids(p).ok(); }

hipError_t launch_attn_win_fwd(const AttnWinArgs& a, int dt, int D, hipStream_t s, bool* sup) {
  if (dt == 1) return fwd_d<_Float16>(a, D, s, sup);
  if (dt == 2) return fwd_d<__bf16>(a, D, s, sup);
  *sup = false;
  return hipErrorInvalidValue;
}

hipError_t launch_attn_win_bwd(const AttnWinArgs& a, int dt, int D, hipStream_t s, bool* sup) {
  if (dt == 1) return bwd_d<_Float16>(a, D, s, sup);
  if (dt == 2) return bwd_d<__bf16>(a, D, s, sup);
  *sup = false;
  return hipErrorInvalidValue;
}

}  // namespace esep
