// A wavefront's query rows against 32 keys of the swizzled K and V tiles, as the walks over pages take them: 32 rows in
// the causal kernels' step (attention_tiles.hpp), or 16 rows on v_mfma_f32_16x16x32, which take half the matrix and
// vector work: what a decoding step of up to 16 query heads to a kv head needs (one row of 700 tokens 11.0 -> 10.1 us, 64 of
// up to 500, 28 / 4 heads 13.8 -> 13.0; where the bytes decide, the same).
//
// Each holds its query rows, the sums and what they belong to: lane's row `row()`, maximum m, sum l (finish() first) and the
// weighted sums, a few columns to a lane.
#pragma once

#include <cmath>

#include "attention_tiles.hpp"

namespace esep {

template <typename T, int D, int ROWS>
struct PagedTile;

template <typename T, int D>
struct PagedTile<T, D, 32> {
  using V8 = typename Mfma<T>::v8;
  int lane;
  V8 q[D / 16];
  f32x16 o[D / 32];
  float m, l;
  __device__ __forceinline__ explicit PagedTile(int lane_) : lane(lane_) {}
  __device__ __forceinline__ int row() const { return lane & 31; }
  // the lane's query row, zeros where there is none
  __device__ __forceinline__ void load(const T* at, bool ok) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) q[c] = ok ? ld16<V8>(at + 16 * c + 8 * (lane >> 5)) : V8{};
#pragma unroll
    for (int md = 0; md < D / 32; ++md) o[md] = f32x16{};
    m = -INFINITY;
    l = 0.f;
  }
  // keys kh .. kh + 31; hides(key): the lane's row does not see it, asked where `some` of the wavefront's do not; none: bits
  // of the halves of 16 keys that nobody sees
  template <class Hides>
  __device__ __forceinline__ void step(const char* ks, const char* vs, float scale_log2, int kh, bool some,
                                       uint32_t none, Hides&& hides) {
    const int hi = lane >> 5;
    fwd_tile_swz<T, D>(ks, vs, lane, scale_log2, q, o, m, l, [&](f32x16& acc) __attribute__((always_inline)) {
      if (some) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (hides(kh + 8 * (i / 4) + 4 * hi + i % 4)) acc[i] = -INFINITY;
      }
      if (none) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (none >> (i / 8) & 1) acc[i] = -INFINITY;
      }
    });
  }
  __device__ __forceinline__ void finish() {}
  __device__ __forceinline__ bool first() const { return lane < 32; }  // of the lanes of a row
  // f(column, four values) of the lane's row
  template <class F>
  __device__ __forceinline__ void each4(F&& f) const {
#pragma unroll
    for (int md = 0; md < D / 32; ++md)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f(32 * md + 8 * j + 4 * (lane >> 5),
          f32x4{o[md][4 * j], o[md][4 * j + 1], o[md][4 * j + 2], o[md][4 * j + 3]});
  }
  __device__ __forceinline__ void store(T* at) const { store_rows_t<T, D>(at, o, lane >> 5, l > 0.f ? 1.f / l : 0.f); }
};

// v_mfma_f32_16x16x32: A[i][k] in lane i + 16 (k / 8), element k % 8; B[k][j] in lane j + 16 (k / 8); C[i][j] in lane j +
// 16 (i / 4), element i % 4.
__device__ __forceinline__ f32x4 mfma16(Mfma<__bf16>::v8 a, Mfma<__bf16>::v8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(Mfma<_Float16>::v8 a, Mfma<_Float16>::v8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// max / sum of a lane's value and lane l ^ 16's, equal in both (as pair_max's of l ^ 32).
__device__ __forceinline__ float quarter_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ __forceinline__ float quarter_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// S^T = K Q^T in two products' rows of 16 keys, lane (j, g = lane / 16) with row j's scores of keys 4 g + i and 16 + 4 g + i;
// O^T += V^T P^T over the 32 keys at once, in the order 4 g + e, 16 + 4 g + e - 4 of P^T's elements e < 8, which is that of
// V^T's two transposing reads. The reference moves by the same rule as in fwd_tile_swz; the sum stays the lane's own until
// finish(). P is rounded to T, the matrix instructions' operand type.
template <typename T, int D>
struct PagedTile<T, D, 16> {
  static constexpr int RB = 2 * D;
  using V8 = typename Mfma<T>::v8;
  int lane;
  uint32_t k0, v0;  // byte offsets of the lane's K row (chunk 0 of its quarter) and of its V rows (columns 0)
  V8 q[D / 32];
  f32x4 o[D / 16];
  float m, l;
  __device__ __forceinline__ explicit PagedTile(int lane_) : lane(lane_) {
    const int j = lane & 15, g = lane >> 4, k = (lane >> 2) & 3, c = lane & 3;
    k0 = (uint32_t)RB * j + 16u * (uint32_t)(g ^ swz<RB>(j));
    v0 = (uint32_t)RB * (4 * g + k) + 16u * (uint32_t)((c >> 1) ^ swz<RB>(4 * g + k)) + 8u * (c & 1);
  }
  __device__ __forceinline__ int row() const { return lane & 15; }
  __device__ __forceinline__ void load(const T* at, bool ok) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) q[c] = ok ? ld16<V8>(at + 32 * c + 8 * (lane >> 4)) : V8{};
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = f32x4{};
    m = -INFINITY;
    l = 0.f;
  }
  // columns 16 d .. of the V tile, transposed: row d + lane % 16 of V^T, the 32 keys in P^T's order
  __device__ __forceinline__ V8 vt(const char* vs, int d) const {
    typedef __attribute__((address_space(3))) s16x4* lds_ptr;
    const uint32_t at = v0 ^ (32u * d);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(vs + at));
    const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(vs + (at + 16u * RB)));
    return __builtin_bit_cast(V8, __builtin_shufflevector(lo, up, 0, 1, 2, 3, 4, 5, 6, 7));
  }
  template <class Hides>
  __device__ __forceinline__ void step(const char* ks, const char* vs, float scale_log2, int kh, bool some,
                                       uint32_t none, Hides&& hides) {
    const int g = lane >> 4;
    f32x4 s[2] = {};
#pragma unroll
    for (int c = 0; c < D / 32; ++c)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = mfma16(ld16<V8>(ks + (k0 ^ (64u * c)) + 16u * RB * t), q[c], s[t]);
    if (some) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (hides(kh + 16 * (i / 4) + 4 * g + i % 4)) s[i / 4][i % 4] = -INFINITY;
    }
    if (none) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (none >> (i / 4) & 1) s[i / 4][i % 4] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i / 4][i % 4]);
    mx = quarter_max(pair_max(mx)) * scale_log2;
    const bool grow = mx > m + 8.f;
    float alpha = 1.f;
    if (grow) {
      alpha = exp2_fast(m - mx);
      m = mx;
    }
    const float nm = m == -INFINITY ? 0.f : -m;
    l *= alpha;
    V8 p;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = exp2_fast(fmaf(s[i / 4][i % 4], scale_log2, nm));
      l += e;
      p[i] = (T)e;
    }
    if (__any(grow)) {
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[d] *= alpha;
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[d] = mfma16(vt(vs, d), p, o[d]);
  }
  __device__ __forceinline__ void finish() { l = quarter_sum(pair_sum(l)); }
  __device__ __forceinline__ bool first() const { return lane < 16; }
  template <class F>
  __device__ __forceinline__ void each4(F&& f) const {
#pragma unroll
    for (int d = 0; d < D / 16; ++d) f(16 * d + 4 * (lane >> 4), o[d]);
  }
  __device__ __forceinline__ void store(T* at) const {
    typedef T v4 __attribute__((ext_vector_type(4)));
    const float inv = l > 0.f ? 1.f / l : 0.f;
    each4([&](int column, f32x4 v) {
      v4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (T)(v[e] * inv);
      *reinterpret_cast<v4*>(at + column) = x;
    });
  }
};

}  // namespace esep
