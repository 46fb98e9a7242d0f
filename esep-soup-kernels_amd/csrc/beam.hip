// Beam search's selection: of the values score_w + logit_{w, t} - lse_w of a request's W beams over the V tokens
// the `keep` greatest, ties to the lowest w V + t, in two launches. A beam is out (all its values -inf) where its
// score or its lse is not finite (no finite logit, a NaN, an infinity above).
//
// The logits are read once. k_beam_rows: a block holds a piece of a row in registers and leaves the piece's maximum,
// its sum of exponentials and its `keep` greatest logits as 64-bit keys (order of the logit, then of the lowest
// token). The greatest of 64 lanes' own maxima are found first, wavefront by wavefront: the keep-th of them
// bounds the piece's keep-th greatest from below, so that only what reaches the highest of these bounds is listed (about
// 2 keep), and a listed key's place is the number of greater ones. k_beam_join: lse of each beam from the pieces'
// parts, the same selection among the pieces' candidates by value, in 64 bits (two beams' values lie closer than 32 bits
// tell apart once in about 10^4 choices). Where ties fill the list the greatest is taken `keep` times instead.
//
// Bound by two launches' latency (one request of 4 beams over 151936 in bf16, keep 8: 4.4 + 4.4 us, where its bytes
// take 0.2), with many rows by the logits and a block's chain from its loads to its list. Both launches, graph
// replays, cold caches, us (the bytes' time): 24 x 5 x 151936 fp32, keep 5 22.6 (14.5), with one beam of five alive
// 13.2 (2.9); 128 x 4 x 151936 bf16, keep 8 44.9 (30.9), without the lists 40; 16 x 8 x 50001 fp32, keep 16 15.9
// (5.1; read an element at a time, as its rows begin anywhere, 25.8); 1 x 8 x 151936 bf16, keep 64 21.9; 64 x 4 x
// 151936 bf16, keep 64 47 (with 64 groups to bound it 517: one list in 50 overflows); 1 x 64 x 151936, keep 64 79:
// 78000 candidates for the join's one block. Loads past the caches change none of it by more than 3%.
#include "beam.hpp"

#include <cmath>

#include "common.hpp"

namespace esep {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kList = 512;

// A float's bits in the order of the floats, -0 as 0 (-inf lowest but for NaN, which does not come here).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp_f<0xB1>(v));
  v = fmaxf(v, dpp_f<0x4E>(v));
  v = fmaxf(v, dpp_f<0x141>(v));
  v = fmaxf(v, dpp_f<0x140>(v));
  const float r0 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 0));
  const float r1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16));
  const float r2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 32));
  const float r3 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 48));
  return fmaxf(fmaxf(r0, r1), fmaxf(r2, r3));
}

// A bound that at least `keep` of the wavefront's 64 G keys reach, and of the values with these first 20 bits the
// greatest: bit by bit, the keys at or above it counted. 0 where fewer are finite.
constexpr int kBoundBits = 20;
template <int G>
__device__ __forceinline__ uint32_t wave_bound(const uint32_t (&key)[G], int keep) {
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 32 - kBoundBits; --bit) {
    const uint32_t t = bound | 1u << bit;
    int n = 0;
#pragma unroll
    for (int i = 0; i < G; ++i) n += __popcll(__ballot(key[i] >= t));
    if (n >= keep) bound = t;
  }
  return bound;
}
// It as a float, at least the lowest finite one.
__device__ __forceinline__ float bound_of(uint32_t key) { return unordered(key < 0x00800000u ? 0x00800000u : key); }
// A bound that the `keep` greatest of what the block's threads have put into v (after a barrier) reach, and the
// greatest of all. The threads make 64 groups, for a large `keep` 256: of 64 the least one's maximum would bound 64
// of them, which 300 values of random rows reach (and more than the list holds in one row of 50), of 256 74 do.
constexpr int kFewKeep = 32;
template <int NW>
__device__ __forceinline__ float block_bound(const float (&v)[NW * 64], int lane, int keep, float* top) {
  float m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = v[64 * i + lane];
#pragma unroll
  for (int i = 4; i < NW; ++i) m[i % 4] = fmaxf(m[i % 4], v[64 * i + lane]);
  const float all = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  *top = wave_max(all);
  if (keep <= kFewKeep) {
    const uint32_t key[1] = {ordered(all)};
    return bound_of(wave_bound(key, keep));
  }
  const uint32_t key[4] = {ordered(m[0]), ordered(m[1]), ordered(m[2]), ordered(m[3])};
  return bound_of(wave_bound(key, keep));
}

// Lanes that count a listed candidate's betters together, and their sum, in each of them.
constexpr int kRankLanes = 8;
__device__ __forceinline__ int rank_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);   // lane ^ 1
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);   // lane ^ 2
  return v + __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false);  // the other quad of each 8
}

// How many of a lane's share of the n listed are better; of a long list four looked at at once (384 in one piece 34 -> 13 us;
// of ten that takes 0.3 us more).
template <class F>
__device__ __forceinline__ int betters(int n, int first, F&& better) {
  int count = 0;
  if (n <= 64) {
    for (int j = first; j < n; j += kRankLanes) count += better(j);
    return count;
  }
  for (int j0 = first; j0 < n; j0 += 4 * kRankLanes) {
    bool b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = better(j0 + i * kRankLanes < n ? j0 + i * kRankLanes : j0);
#pragma unroll
    for (int i = 0; i < 4; ++i) count += b[i] && j0 + i * kRankLanes < n;
  }
  return count;
}

// 16 bytes of logits, wherever they lie (a row of an odd vocabulary begins anywhere).
typedef uint32_t Any16 __attribute__((ext_vector_type(4), aligned(2)));

// The piece's elements of thread i: i * 8 .. + 7 of each run of 2048, whatever the row's alignment, so that equal
// rows give equal sums. (Registers for six wavefronts to a SIMD: 128 requests of 4 beams over 151936 in bf16 47.7 ->
// 44.9 us, where the compiler's own choice leaves five, and eight spill: 48.5. With six, at U = 4, three registers go to
// scratch memory behind the branch of a list that overflows, none before it.)
template <typename T, int U>
__global__ __launch_bounds__(kBeamThreads, 6) void k_beam_rows(const BeamArgs a) {
  constexpr int NW = kBeamThreads / 64;
  __shared__ float w_sum[NW], best[kBeamThreads];
  __shared__ uint64_t list[kList];
  __shared__ uint64_t w_best[NW];
  __shared__ int count;
  const int row = blockIdx.y, split = blockIdx.x, lane = threadIdx.x & 63, w = wave_id();
  const float score = a.scores[row];
  if (!(fabsf(score) < INFINITY)) return;  // the beam is out: the join does not look at its pieces
  const int r = row / a.W;
  const T* x = static_cast<const T*>(a.logits) + r * a.r_bs + (row - r * a.W) * a.w_bs;
  const int base = split * a.each + 8 * (int)threadIdx.x;
  const int end = base - 8 * (int)threadIdx.x + a.each < a.V ? base - 8 * (int)threadIdx.x + a.each : a.V;
  float v[U][8];
  if (threadIdx.x == 0) count = 0;
  // all of it is asked for at once, in pieces of 16 bytes at any address; eights that the row does not fill are read at its
  // begin (or not: it has fewer) and replaced
  Raw<T> raw[U];
  if (a.V >= 8) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Any16* at = reinterpret_cast<const Any16*>(x + (base + 2048 * u + 7 < end ? base + 2048 * u : 0));
      raw[u].a = at[0];
      if constexpr (sizeof(T) == 4) raw[u].b = at[1];
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = Raw<T>{};
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    Buf<T>::unpack(raw[u], v[u]);
    const int at = base + 2048 * u;
    if (at + 7 >= end) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = -INFINITY;
      if (at < end) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (at + e < end) v[u][e] = (float)x[at + e];
      }
    }
  }
  float mine = -INFINITY, run[U];  // the greatest of all, of each eight; NaN is passed over
#pragma unroll
  for (int u = 0; u < U; ++u) {
    run[u] = v[u][0];
#pragma unroll
    for (int e = 1; e < 8; ++e) run[u] = fmaxf(run[u], v[u][e]);
    mine = fmaxf(mine, run[u]);
  }
  best[threadIdx.x] = mine;
  __syncthreads();
  float top;
  const float bound = block_bound<NW>(best, lane, a.keep, &top);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += __builtin_amdgcn_exp2f((v[u][e] - ref) * kLog2e);
  sum = wave_sum(sum);
  if (lane == 0) w_sum[w] = sum;
  auto key = [&](int u, int e) {
    return (uint64_t)ordered(v[u][e]) << 32 | (uint32_t)~(base + 2048 * u + e);
  };
  if (mine >= bound) {
    int n = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (run[u] >= bound) {
#pragma unroll
        for (int e = 0; e < 8; ++e) n += v[u][e] >= bound;
      }
    int at = atomicAdd(&count, n);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (run[u] >= bound) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v[u][e] >= bound) {
            if (at < kList) list[at] = key(u, e);
            ++at;
          }
      }
  }
  __syncthreads();
  const int64_t part = (int64_t)row * a.splits + split;
  if (threadIdx.x == 0) {
    float all = w_sum[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) all += w_sum[i];
    a.stat[part] = make_float2(top, all);
  }
  uint64_t* out = a.cand + part * a.keep;
  const int n = count;
  if (n <= kList) {
    for (int i = threadIdx.x / kRankLanes; i < n; i += kBeamThreads / kRankLanes) {
      const uint64_t k = list[i];
      const int place = rank_sum(betters(n, (int)threadIdx.x % kRankLanes, [&](int j) { return list[j] > k; }));
      if (place < a.keep && threadIdx.x % kRankLanes == 0) out[place] = k;
    }
    for (int i = n + threadIdx.x; i < a.keep; i += kBeamThreads) out[i] = 0;
    return;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.keep; ++k) {  // at least kList > keep candidates
    uint64_t best = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint64_t at = key(u, e);
        if (v[u][e] > -INFINITY && at < last && at > best) best = at;
      }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const uint64_t o = __shfl_xor(best, d);
      best = o > best ? o : best;
    }
    if (lane == 0) w_best[w] = best;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) best = w_best[i] > best ? w_best[i] : best;
    if (threadIdx.x == 0) out[k] = best;
    last = best;
    __syncthreads();
  }
}

// A candidate of the join: its value and its place w V + t; the greater value first, then the lower place. None: -inf
// at a place that no candidate has.
struct Cand {
  double value;
  int at;
};
constexpr int kNoPlace = 0x7fffffff;
__device__ __forceinline__ bool before(const Cand& x, const Cand& y) {
  return x.value > y.value || (x.value == y.value && x.at < y.at);
}

constexpr int kJoinFirst = kBeamJoinFirst, kJoinMore = 8, kJoinMostBeams = 64;

template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_beam_join(const BeamArgs a) {
  constexpr int NW = THREADS / 64;
  // lse = top + rest, apart, so that large logits do not swallow the rest; score: NaN where the beam is out
  __shared__ double rest[kJoinMostBeams], score[kJoinMostBeams];
  __shared__ float tops[kJoinMostBeams];
  __shared__ Cand list[kList], w_best[NW];
  __shared__ float group[THREADS];
  __shared__ int chosen[kBeamMostKeep];
  __shared__ int count;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = wave_id();
  const int per = a.splits * a.keep, all = a.W * per;
  const uint64_t* keys = a.cand + (int64_t)r * all;
  // Candidate j of the thread: each 64 of them turned by one lane more, as a piece's lie there in their order, and 64 groups
  // of lanes of which some hold the pieces' first and others their last would bound nothing.
  auto index = [&](int j) {
    const int chunk = j * NW + w;
    return 64 * chunk + ((lane + chunk) & 63);
  };
  // everything is asked for at once: the thread's first candidates, the pieces' parts (those of a beam that is out hold
  // nothing, and are not used)
  uint64_t key[kJoinFirst];
#pragma unroll
  for (int j = 0; j < kJoinFirst; ++j) key[j] = index(j) < all ? keys[index(j)] : 0;
  if (tid == 0) count = 0;
#pragma unroll 1
  for (int b = w; b < a.W; b += NW) {
    const int row = r * a.W + b;
    const float sc = a.scores[row];
    const float2* st = a.stat + (int64_t)row * a.splits;
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 p0 = lane < a.splits ? st[lane] : none, p1 = lane + 64 < a.splits ? st[lane + 64] : none;
    double l = 0.0;
    float top = fmaxf(p0.x, p1.x);
    const bool in = fabsf(sc) < INFINITY;
    if (in) {
#pragma unroll 1
      for (int i = lane + 128; i < a.splits; i += 64) top = fmaxf(top, st[i].x);
      top = wave_max(top);
      auto part = [&](const float2& p) {  // a piece without a finite logit has 0, or a NaN
        return p.x == -INFINITY ? p.y : p.y * __builtin_amdgcn_exp2f((p.x - top) * kLog2e);
      };
      double sum = (double)part(p0) + (double)part(p1);
#pragma unroll 1
      for (int i = lane + 128; i < a.splits; i += 64) sum += (double)part(st[i]);
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
      l = log(sum);
    }
    if (lane == 0) {
      tops[b] = top;
      rest[b] = l;
      score[b] = in && fabsf(top) < INFINITY && fabs(l) < (double)INFINITY ? (double)sc : (double)NAN;
    }
  }
  __syncthreads();
  auto value = [&](int i, uint64_t k) {  // of candidate i
    const int b = i / per;
    if (k == 0 || !(score[b] == score[b])) return Cand{-(double)INFINITY, kNoPlace};
    return Cand{(((double)unordered((uint32_t)(k >> 32)) - (double)tops[b]) - rest[b]) + score[b],
                b * a.V + (int)~(uint32_t)k};
  };
  // A value in 32 bits, in the values' order: a quarter of it, as three of fp32's greatest may be taken from 0 (score, and a
  // logit far below its row's greatest), and what rounds to -inf would count as none.
  auto in32 = [](const Cand& c) { return (float)(0.25 * c.value); };
  Cand mine[kJoinFirst];
  float best32 = -INFINITY;
#pragma unroll
  for (int j = 0; j < kJoinFirst; ++j) {
    mine[j] = value(index(j) < all ? index(j) : 0, key[j]);
    best32 = fmaxf(best32, in32(mine[j]));
  }
  const int rounds = (all + THREADS - 1) / THREADS;
  // f of the thread's candidates from j0 on, kJoinMore asked for at once
  auto each_from = [&](int j0, auto&& f) {
#pragma unroll 1
    for (int j = j0; j < rounds; j += kJoinMore) {
      uint64_t more[kJoinMore];
#pragma unroll
      for (int i = 0; i < kJoinMore; ++i) more[i] = index(j + i) < all ? keys[index(j + i)] : 0;
#pragma unroll
      for (int i = 0; i < kJoinMore; ++i) f(value(index(j + i) < all ? index(j + i) : 0, more[i]));
    }
  };
  each_from(kJoinFirst, [&](const Cand& c) { best32 = fmaxf(best32, in32(c)); });
  group[tid] = best32;
  __syncthreads();
  float highest;
  const float bound = block_bound<NW>(group, lane, a.keep, &highest);
  // what reaches the bound
  auto enter = [&](const Cand& c) {
    if (in32(c) >= bound) {
      const int at = atomicAdd(&count, 1);
      if (at < kList) list[at] = c;
    }
  };
#pragma unroll
  for (int j = 0; j < kJoinFirst; ++j) enter(mine[j]);
  if (best32 >= bound) each_from(kJoinFirst, enter);
  __syncthreads();
  auto put = [&](int place, const Cand& c) {
    const int o = r * a.keep + place, b = c.at / a.V;
    a.out_scores[o] = (float)c.value;
    a.out_parents[o] = b;
    a.out_tokens[o] = c.at - b * a.V;
    chosen[place] = c.at;
  };
  const int n = count;
  if (n > kList) {  // ties: the greatest, `keep` times
    Cand last{(double)INFINITY, -1};
#pragma unroll 1
    for (int k = 0; k < a.keep; ++k) {
      Cand best{-(double)INFINITY, kNoPlace};
      each_from(0, [&](const Cand& c) {
        if (before(last, c) && before(c, best)) best = c;
      });
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        const Cand o{__shfl_xor(best.value, d), __shfl_xor(best.at, d)};
        if (before(o, best)) best = o;
      }
      if (lane == 0) w_best[w] = best;
      __syncthreads();
#pragma unroll 1
      for (int i = 0; i < NW; ++i)
        if (before(w_best[i], best)) best = w_best[i];
      if (tid == 0) put(k, best);
      last = best;
      __syncthreads();
    }
    return;
  }
  for (int i = tid / kRankLanes; i < n; i += THREADS / kRankLanes) {
    const Cand c = list[i];
    const int place = rank_sum(betters(n, tid % kRankLanes, [&](int j) { return before(list[j], c); }));
    if (place < a.keep && tid % kRankLanes == 0) put(place, c);
  }
  if (n >= a.keep) return;
  // the others are -inf, at the lowest places that are not among the chosen
  __syncthreads();
  if (tid != 0) return;
  int at = 0;
#pragma unroll 1
  for (int k = n; k < a.keep; ++at) {
    bool taken = false;
#pragma unroll 1
    for (int j = 0; j < n; ++j) taken |= chosen[j] == at;
    if (!taken) put(k++, Cand{-(double)INFINITY, at});
  }
}

template <typename T>
hipError_t run(const BeamArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)a.splits, (unsigned)(a.R * a.W));
  if (a.piece == 2048)
    hipLaunchKernelGGL((k_beam_rows<T, 1>), grid, dim3(kBeamThreads), 0, s, a);
  else if (a.piece == 4096)
    hipLaunchKernelGGL((k_beam_rows<T, 2>), grid, dim3(kBeamThreads), 0, s, a);
  else
    hipLaunchKernelGGL((k_beam_rows<T, 4>), grid, dim3(kBeamThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // small blocks for many requests' few candidates (2000 of 24 candidates 41.5 -> 32.5 us in all, 4000 of 32 90 -> 72; 24 of
  // 475 13.2 -> 13.6)
  if (a.R > 256 && (int64_t)a.W * a.splits * a.keep <= 256 * kJoinFirst)
    hipLaunchKernelGGL((k_beam_join<256>), dim3((unsigned)a.R), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((k_beam_join<1024>), dim3((unsigned)a.R), dim3(1024), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_beam_select(const BeamArgs& a, int dt, hipStream_t s, bool* sup) {
  *sup = true;
  if (dt == 0) return run<float>(a, s);
  if (dt == 1) return run<_Float16>(a, s);
  if (dt == 2) return run<__bf16>(a, s);
  *sup = false;
  return hipErrorInvalidValue;
}

}  // namespace esep
