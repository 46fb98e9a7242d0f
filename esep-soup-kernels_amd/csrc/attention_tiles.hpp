// One step of each attention kernel: a wavefront's 32 queries against 32 keys held in swizzled LDS tiles
// (attention.hpp: SwzFill, swz_row_base, SwzTr). The kernels differ in which tiles they walk and in
// what a query sees, which comes in as `mask`.
#pragma once

#include <cmath>

#include "attention.hpp"

namespace esep {

constexpr float kLog2e = 1.4426950408889634f;

// Keys after the lane's query qi: score element i belongs to key kh + 8 (i / 4) + 4 hi + i % 4. Only where
// the 32 keys reach past the wavefront's first query qw0.
__device__ __forceinline__ void mask_future(f32x16& acc, int kh, int qw0, int qi, int hi) {
  if (kh + 31 > qw0) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int kj = kh + 8 * (i / 4) + 4 * hi + (i % 4);
      if (kj > qi) acc[i] = -INFINITY;
    }
  }
}

// Keys past `top`, or at `low` and before it but no sinks. Only where a border crosses the 32 keys: utop
// is the least top and ulow the greatest low of the wavefront.
__device__ __forceinline__ void mask_window(f32x16& acc, int kh, int utop, int ulow, int top, int low,
                                            int sink_hi, int hi) {
  if (kh + 31 > utop || kh <= ulow) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int kj = kh + 8 * (i / 4) + 4 * hi + (i % 4);
      if (kj > top || (kj <= low && kj >= sink_hi)) acc[i] = -INFINITY;
    }
  }
}

// 32 keys of the online softmax for a wavefront's 32 queries: keys kh .. kh + 31, held in 32 rows of
// the swizzled LDS tiles at ks / vs (the layout, its DMA and its readers are in attention.hpp).
// Lane (lq, hi) gets the scores of its query qi against keys kh + 8 (i / 4) + 4 hi + i % 4, i < 16,
// from S^T = K Q^T (K rows from LDS as the A operand, the wave's Q^T in registers as B), then
// updates (m, l) and O^T += V^T P^T, the contraction in the permuted key order of pb (element e of
// chunk c2 is key kh + 16 c2 + 8 (e / 4) + 4 hi + e % 4).
//
// Online softmax (base 2) with a lazy reference: the lane's m moves only when the 32 keys' maximum
// exceeds it by more than 8, so p <= 2^8 (exact in bf16 / fp16 relative terms) and O, l are
// rescaled only where some lane's m moved. Operands are read ahead of their MFMAs (K three, V^T two,
// the first V^T ones before the softmax, whose VALU work hides their latency), pinned by
// scheduling barriers: the compiler sinks each read to just before its use (config 5 forward
// 2.03 -> 1.93 ms).
// The probabilities are rounded to T, the matrix instructions' operand type, before P V (half a step of each; l
// adds them up unrounded): with V and the result in T too, o is off by up to about twice its own rounding.
// mask(acc) sets the scores that the lane's query does not see to -inf.
template <typename T, int D, class Mask>
__device__ __forceinline__ void fwd_tile_swz(const char* ks, const char* vs, int lane,
                                             float scale_log2,
                                             const typename Mfma<T>::v8 (&qb)[D / 16],
                                             f32x16 (&oacc)[D / 32], float& m, float& l,
                                             Mask&& mask) {
  constexpr int RB = 2 * D;
  using V8 = typename Mfma<T>::v8;
  // The MFMA runs go at raised wave priority, the softmax between them at the normal one: with
  // several wavefronts per SIMD the arbiter then feeds the matrix core from a wavefront in its
  // MFMA run ahead of another's vector work (all three kernels; config 5: forward 1.44 -> 1.43
  // ms, backward 5.00 -> 4.91 ms).
  __builtin_amdgcn_s_setprio(1);
  f32x16 acc = f32x16{};
  const uint32_t k0 = swz_row_base<RB>(lane);
  constexpr int KA = 3;
  V8 kbuf[KA];
#pragma unroll
  for (int c = 0; c < KA; ++c) kbuf[c] = ld16<V8>(ks + (k0 ^ (32u * c)));
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    acc = Mfma<T>::run(kbuf[c % KA], qb[c], acc);
    if (c + KA < D / 16) kbuf[c % KA] = ld16<V8>(ks + (k0 ^ (32u * (c + KA))));
    __builtin_amdgcn_sched_barrier(0);
  }
  // V^T operand j: rows 16 (j & 1) .., columns 32 (j >> 1) .. of the V tile
  const SwzTr<RB> vt(lane);
  auto ldv = [&](int j) { return vt.template read<V8>(vs, 16 * (j & 1), j >> 1); };
  constexpr int VA = 2;
  V8 vbuf[VA];
#pragma unroll
  for (int j = 0; j < VA; ++j) vbuf[j] = ldv(j);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_setprio(0);
  mask(acc);
  float mx = acc[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) mx = fmaxf(mx, acc[i]);
  mx = pair_max(mx) * scale_log2;
  const bool grow = mx > m + 8.f;
  float alpha = 1.f;
  if (grow) {
    alpha = exp2_fast(m - mx);
    m = mx;
  }
  const float nm = m == -INFINITY ? 0.f : -m;
  float ps = 0.f;
  V8 pb[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float p = exp2_fast(fmaf(acc[i], scale_log2, nm));
    ps += p;
    pb[i / 8][i % 8] = (T)p;
  }
  ps = pair_sum(ps);
  l = fmaf(l, alpha, ps);
  if (__any(grow)) {
#pragma unroll
    for (int md = 0; md < D / 32; ++md) oacc[md] *= alpha;
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    oacc[j / 2] = Mfma<T>::run(vbuf[j % VA], pb[j % 2], oacc[j / 2]);
    if (j + VA < D / 16) vbuf[j % VA] = ldv(j + VA);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

// 32 keys of the dQ walk for a wavefront's 32 queries: keys kh .. kh + 31, held in 32 rows of the
// swizzled LDS tiles at ks / vs (attention.hpp: SwzFill, swz_row_base, SwzTr). S^T = K Q^T and
// dP^T = V dO^T with the wave's Q and dO as B operands, dS^T = P^T * (dP^T - delta), then
// dQ^T += K^T dS^T with K^T read transposed out of ks and dS^T in the permuted key order. K and V
// operands are read three ahead of their MFMAs and the first two K^T ones before the exponentials
// (config 5 bwd 7.11 -> 6.97 ms). dS is rounded to T, the matrix instructions' operand type.
template <typename T, int D, class Mask>
__device__ __forceinline__ void dq_tile_swz(const char* ks, const char* vs, int lane,
                                            float scale_log2, float lse2, float delta,
                                            const typename Mfma<T>::v8 (&qb)[D / 16],
                                            const typename Mfma<T>::v8 (&db)[D / 16],
                                            f32x16 (&dqa)[D / 32], Mask&& mask) {
  constexpr int RB = 2 * D;
  using V8 = typename Mfma<T>::v8;
  __builtin_amdgcn_s_setprio(1);  // MFMA runs at raised priority, as in the forward
  f32x16 s = f32x16{}, dp = f32x16{};
  const uint32_t r0 = swz_row_base<RB>(lane);
  constexpr int KA = 3;
  V8 kbuf[KA], vbuf[KA];
#pragma unroll
  for (int c = 0; c < KA; ++c) {
    kbuf[c] = ld16<V8>(ks + (r0 ^ (32u * c)));
    vbuf[c] = ld16<V8>(vs + (r0 ^ (32u * c)));
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    s = Mfma<T>::run(kbuf[c % KA], qb[c], s);
    dp = Mfma<T>::run(vbuf[c % KA], db[c], dp);
    if (c + KA < D / 16) {
      kbuf[c % KA] = ld16<V8>(ks + (r0 ^ (32u * (c + KA))));
      vbuf[c % KA] = ld16<V8>(vs + (r0 ^ (32u * (c + KA))));
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  const SwzTr<RB> kt(lane);
  constexpr int TA = 2;
  V8 tbuf[TA];
#pragma unroll
  for (int j = 0; j < TA; ++j) tbuf[j] = kt.template read<V8>(ks, 16 * (j & 1), j >> 1);
  __builtin_amdgcn_sched_barrier(0);
  mask(s);
  __builtin_amdgcn_s_setprio(0);
  V8 dsb[2];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float p = exp2_fast(fmaf(s[i], scale_log2, -lse2));
    dsb[i / 8][i % 8] = (T)(p * (dp[i] - delta));
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    dqa[j / 2] = Mfma<T>::run(tbuf[j % TA], dsb[j % 2], dqa[j / 2]);
    if (j + TA < D / 16) tbuf[j % TA] = kt.template read<V8>(ks, 16 * ((j + TA) & 1), (j + TA) >> 1);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

}  // namespace esep
