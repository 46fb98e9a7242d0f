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
#include "beam.hpp"

#include <cmath>

#include "common.hpp"

namespace esep {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kList = 512;

// A float's bits in the order of the floats (-inf lowest but for NaN, which does not come here).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x);
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

// A bound that at least `keep` of the wavefront's lanes reach with v; -inf where fewer have more than that.
__device__ __forceinline__ float wave_bound(float v, int keep) {
  int n = 0;
  float bound = -INFINITY;
  while (n < keep) {
    bound = wave_max(v);
    if (bound == -INFINITY) break;
    const uint64_t at = __ballot(v == bound);
    n += (int)__popcll(at);
    if (v == bound) v = -INFINITY;
  }
  return bound;
}

// The piece's elements of thread i: i * 8 .. + 7 of each run of 2048, whatever the row's alignment, so that equal
// rows give equal sums.
template <typename T, int U, bool VEC>
__global__ __launch_bounds__(kBeamThreads) void k_beam_rows(const BeamArgs a) {
  constexpr int NW = kBeamThreads / 64;
  __shared__ float w_max[NW], w_sum[NW], w_bound[NW];
  __shared__ uint64_t list[kList];
  __shared__ uint64_t w_best[NW];
  __shared__ int count;
  const int row = blockIdx.y, split = blockIdx.x, lane = threadIdx.x & 63, w = wave_id();
  const float score = a.scores[row];
  if (!(fabsf(score) < INFINITY)) return;  // the beam is out: the join does not look at its pieces
  const int r = row / a.W;
  const T* x = static_cast<const T*>(a.logits) + r * a.r_bs + (row - r * a.W) * a.w_bs;
  const int base = split * a.piece + 8 * (int)threadIdx.x;
  float v[U][8];
  if (threadIdx.x == 0) count = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = base + 2048 * u;
    if constexpr (VEC) {
      if (i < a.V) {  // whole: V is a multiple of 8
        Chunk<T>::load(x + i, v[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[u][e] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = i + e < a.V ? (float)x[i + e] : -INFINITY;
    }
  }
  float mine = -INFINITY;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) mine = fmaxf(mine, v[u][e]);  // NaN is passed over
  const float wm = wave_max(mine);
  const float wb = wave_bound(mine, a.keep);
  if (lane == 0) {
    w_max[w] = wm;
    w_bound[w] = wb;
  }
  __syncthreads();
  float top = w_max[0], bound = w_bound[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) top = fmaxf(top, w_max[i]), bound = fmaxf(bound, w_bound[i]);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += __builtin_amdgcn_exp2f((v[u][e] - ref) * kLog2e);
  sum = wave_sum(sum);
  if (lane == 0) w_sum[w] = sum;
  auto key = [&](int u, int e) {  // -0 counts as 0
    const float f = v[u][e] == 0.f ? 0.f : v[u][e];
    return (uint64_t)ordered(f) << 32 | (uint32_t)~(base + 2048 * u + e);
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (v[u][e] >= bound && v[u][e] > -INFINITY) {
        const int at = atomicAdd(&count, 1);
        if (at < kList) list[at] = key(u, e);
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
    for (int i = threadIdx.x; i < n; i += kBeamThreads) {
      const uint64_t k = list[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += list[j] > k;
      if (place < a.keep) out[place] = k;
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

// A candidate of the join: its value and its place w V + t; the greater value first, then the lower place.
struct Cand {
  double value;
  int64_t at;
};
__device__ __forceinline__ bool before(const Cand& x, const Cand& y) {
  return x.value > y.value || (x.value == y.value && x.at < y.at);
}

constexpr int kJoinThreads = 1024, kJoinMostBeams = 64;

__global__ __launch_bounds__(kJoinThreads) void k_beam_join(const BeamArgs a) {
  constexpr int NW = kJoinThreads / 64;
  // lse = top + rest, apart, so that large logits do not swallow the rest; score: NaN where the beam is out
  __shared__ double rest[kJoinMostBeams], score[kJoinMostBeams];
  __shared__ float tops[kJoinMostBeams];
  __shared__ Cand list[kList], w_best[NW];
  __shared__ float w_bound[NW];
  __shared__ int64_t chosen[kBeamMostKeep];
  __shared__ int count, found;
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = wave_id();
  if (threadIdx.x == 0) count = 0, found = 0;
  for (int b = w; b < a.W; b += NW) {
    const int64_t row = (int64_t)r * a.W + b;
    const float sc = a.scores[row];
    double l = 0.0;
    float top = -INFINITY;
    const bool in = fabsf(sc) < INFINITY;
    if (in) {
      const float2* st = a.stat + row * a.splits;
      for (int i = lane; i < a.splits; i += 64) top = fmaxf(top, st[i].x);
      top = wave_max(top);
      double sum = 0.0;
      for (int i = lane; i < a.splits; i += 64) {
        const float2 p = st[i];
        sum += p.x == -INFINITY ? (double)p.y : (double)p.y * exp((double)p.x - (double)top);
      }
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
  const int per = a.splits * a.keep, all = a.W * per;
  const uint64_t* keys = a.cand + (int64_t)r * all;
  auto get = [&](int i, Cand& c) {  // whether there is one
    const int b = i / per;
    if (!(score[b] == score[b])) return false;
    const uint64_t k = keys[i];
    if (k == 0) return false;
    c.value = (((double)unordered((uint32_t)(k >> 32)) - (double)tops[b]) - rest[b]) + score[b];
    c.at = (int64_t)b * a.V + (int64_t)(uint32_t)~(uint32_t)k;
    return true;
  };
  float mine = -INFINITY;
  for (int i = threadIdx.x; i < all; i += kJoinThreads) {
    Cand c;
    if (get(i, c)) mine = fmaxf(mine, (float)c.value);
  }
  const float wb = wave_bound(mine, a.keep);
  if (lane == 0) w_bound[w] = wb;
  __syncthreads();
  float bound = w_bound[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) bound = fmaxf(bound, w_bound[i]);
  // by value in 32 bits (rounding keeps the order): what reaches the bound
  for (int i = threadIdx.x; i < all; i += kJoinThreads) {
    Cand c;
    if (get(i, c) && (float)c.value >= bound) {
      const int at = atomicAdd(&count, 1);
      if (at < kList) list[at] = c;
    }
  }
  __syncthreads();
  auto put = [&](int place, const Cand& c) {
    const int64_t o = (int64_t)r * a.keep + place;
    const int b = (int)(c.at / a.V);
    a.out_scores[o] = (float)c.value;
    a.out_parents[o] = b;
    a.out_tokens[o] = (int)(c.at - (int64_t)b * a.V);
    chosen[place] = c.at;
  };
  const int n = count;
  if (n <= kList) {
    for (int i = threadIdx.x; i < n; i += kJoinThreads) {
      const Cand c = list[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += before(list[j], c);
      if (place < a.keep) put(place, c);
    }
    if (threadIdx.x == 0) found = n < a.keep ? n : a.keep;
  } else {
    Cand last{(double)INFINITY, -1};
    for (int k = 0; k < a.keep; ++k) {
      Cand best{-(double)INFINITY, INT64_MAX};
      for (int i = threadIdx.x; i < all; i += kJoinThreads) {
        Cand c;
        if (get(i, c) && before(last, c) && before(c, best)) best = c;
      }
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        const Cand o{__shfl_xor(best.value, d), __shfl_xor(best.at, d)};
        if (before(o, best)) best = o;
      }
      if (lane == 0) w_best[w] = best;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NW; ++i)
        if (before(w_best[i], best)) best = w_best[i];
      if (threadIdx.x == 0) put(k, best);
      last = best;
      __syncthreads();
    }
    if (threadIdx.x == 0) found = a.keep;
  }
  __syncthreads();
  // fewer than `keep`: the others are -inf, the lowest places that are not among the chosen
  const int f = found;
  if (f < a.keep && threadIdx.x == 0) {
    int64_t at = 0;
    for (int k = f; k < a.keep; ++at) {
      bool taken = false;
      for (int j = 0; j < f; ++j) taken |= chosen[j] == at;
      if (taken) continue;
      put(k, Cand{-(double)INFINITY, at});
      ++k;
    }
  }
}

template <typename T, int U>
void rows(const BeamArgs& a, bool vec, hipStream_t s) {
  const dim3 grid((unsigned)a.splits, (unsigned)(a.R * a.W));
  if (vec)
    hipLaunchKernelGGL((k_beam_rows<T, U, true>), grid, dim3(kBeamThreads), 0, s, a);
  else
    hipLaunchKernelGGL((k_beam_rows<T, U, false>), grid, dim3(kBeamThreads), 0, s, a);
}

template <typename T>
hipError_t run(const BeamArgs& a, bool vec, hipStream_t s) {
  if (a.piece == 2048)
    rows<T, 1>(a, vec, s);
  else if (a.piece == 4096)
    rows<T, 2>(a, vec, s);
  else
    rows<T, 4>(a, vec, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_beam_join, dim3((unsigned)a.R), dim3(kJoinThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_beam_select(const BeamArgs& a, int dt, bool vec, hipStream_t s, bool* sup) {
  *sup = true;
  if (dt == 0) return run<float>(a, vec, s);
  if (dt == 1) return run<_Float16>(a, vec, s);
  if (dt == 2) return run<__bf16>(a, vec, s);
  *sup = false;
  return hipErrorInvalidValue;
}

}  // namespace esep
