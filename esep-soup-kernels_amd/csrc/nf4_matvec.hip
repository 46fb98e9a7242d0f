// Products of a few rows (up to 16) with NF4 weights: y[m][n] = sum_k x[m][k] W[n][k] (+ bias[n]), W decoded in
// registers and never written. W[n][k] = nf4[nibble] * scale, the scale of 64 consecutive elements from its 8-bit
// store as in nf4.hip.
//
// Bound by the packed bytes (half a byte per weight and 1 / 64 for the scales), and below a few MB by the launch
// and one trip to memory. At those bytes' rate a CU has about 5 cycles for 64 weights, so the decode decides:
//   - a byte's two codes come from one LDS read of a table of 256 pairs in x's type, 32 copies of it, one to a
//     bank, so that 64 lanes read without conflicts (two VALU instructions and one LDS read per two weights);
//   - the products run on v_mfma_f32_16x16x32, x as the A operand and 16 rows of W as B: the contraction over
//     lanes costs no shuffles, and up to 8 rows of x cost what one does;
//   - the scales multiply sums, not weights: 16 bytes of a W row are half a scale block, so lanes (n, q = 0, 1) hold
//     one block and (n, q = 2, 3) the next. A's 16 rows are 8 rows of x twice, the first with zeros against
//     q = 2, 3, the second against q = 0, 1, so that each of D's values belongs to one block, whose scale is
//     that of the lane that holds it. Four products of 128 k are then added with one fma per value.
// The codes are rounded to x's type (fp16 2^-12, bf16 2^-9 relative at most on average half of that), as
// dequantize_nf4 rounds the whole weight to it; scales, products and sums stay in fp32.
//
// A wavefront takes 16 rows of W and a share of k (KS shares, added through LDS in their order); blocks of 8
// wavefronts walk groups of 8 / KS tiles.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "nf4.hpp"

namespace esep {
namespace {

constexpr int kMvThreads = 512, kMvWaves = 8;

template <typename T>
struct Mv;
template <>
struct Mv<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mv<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ f32x4 run(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

__device__ __forceinline__ float mv_scale(float c, float a2, float off) {
#pragma clang fp contract(off)
  const float prod = c * a2;  // two roundings, as the format's decoder
  return prod + off;
}

template <typename T>
__device__ __forceinline__ uint32_t mv_pair(float a, float b) {
  typedef T v2 __attribute__((ext_vector_type(2)));
  const v2 p = {(T)a, (T)b};
  return __builtin_bit_cast(uint32_t, p);
}

// What a wavefront needs of 128 k: 16 bytes of its lane's row, x, the block's scale.
template <int MT>
struct MvStage {
  uint4 w;
  uint4 x[MT][4];
  uint8_t am;
  float a2;
};

template <typename T, int MT, int KS>
__global__ __launch_bounds__(kMvThreads, MT == 1 ? 4 : 2) void k_nf4_matvec(const Nf4MvArgs a) {
  constexpr int TPB = kMvWaves / KS;
  using V8 = typename Mv<T>::v8;
  __shared__ __align__(16) uint32_t tab[256 * 32];
  __shared__ float code2[256];
  __shared__ float red[KS > 1 ? 2 : 1][KS > 1 ? kMvWaves : 1][MT * 8][16];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ks = wave % KS, ti = wave / KS;
  const int lq = lane & 15, q = lane >> 4;
  const int KB = a.K / 64, steps = (KB + 1) / 2;
  const int s0 = steps * ks / KS, s1 = steps * (ks + 1) / KS;
  // x: this lane's row of each 8, read only against its own block's lanes
  const bool mine = (q >> 1) == (lq >> 3);
  const T* xp[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    xp[t] = static_cast<const T*>(a.x) + (int64_t)(8 * t + (lq & 7)) * a.ldx + 32 * q;
  const uint32_t copy = 4 * (lane & 31);
  const char* tabb = reinterpret_cast<const char*>(tab);

  int cur = -1, buf = 0;
  float off = 0.f;
  for (int grp = blockIdx.x; grp < a.groups; grp += gridDim.x) {
    int wi = 0;
    while (wi + 1 < a.n && grp >= a.w[wi + 1].group0) ++wi;
    const Nf4MvWeight& w = a.w[wi];
    const int row = ((grp - w.group0) * TPB + ti) * 16 + lq;
    const int rc = row < w.N ? row : w.N - 1;
    const char* wp = static_cast<const char*>(w.packed) + (int64_t)rc * KB * 32 + 16 * q;
    const int64_t f0 = (int64_t)rc * KB + (lane >> 5);

    auto load = [&](MvStage<MT>& st, int s) {
      const bool ok = 2 * s + (q >> 1) < KB;
      st.w = ok ? *reinterpret_cast<const uint4*>(wp + 64 * (int64_t)s) : make_uint4(0, 0, 0, 0);
      st.am = ok ? w.absmax[f0 + 2 * s] : 0;
      st.a2 = ok ? w.absmax2[(f0 + 2 * s) >> 8] : 0.f;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const bool in = ok && mine && 8 * t + (lq & 7) < a.M;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st.x[t][i] = in ? *reinterpret_cast<const uint4*>(xp[t] + 128 * s + 8 * i)
                          : make_uint4(0, 0, 0, 0);
      }
    };
    f32x4 tot[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) tot[t] = f32x4{};
    MvStage<MT> st[2];
    if (s0 < s1) load(st[0], s0);
    if (s0 + 1 < s1) load(st[1], s0 + 1);

    if (wi != cur) {  // the weight's tables, while its first bytes are on their way
      if (cur >= 0) __syncthreads();
      cur = wi;
      off = *w.offset;
      const float code = w.nf4[lane & 15];
      for (int i = tid; i < 256 * 8; i += kMvThreads) {
        const int e = i / 8;
        const uint32_t p = mv_pair<T>(__shfl(code, e >> 4), __shfl(code, e & 15));
        reinterpret_cast<uint4*>(tab)[i] = make_uint4(p, p, p, p);
      }
      if (tid < 256) code2[tid] = w.code2[tid];
      __syncthreads();
    }

    auto comp = [&](const MvStage<MT>& st, int s) {
      f32x4 acc[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = f32x4{};
      const uint32_t wd[4] = {st.w.x, st.w.y, st.w.z, st.w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 b;
        b.x = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] << 7) & 0x7f80u) | copy));
        b.y = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] >> 1) & 0x7f80u) | copy));
        b.z = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] >> 9) & 0x7f80u) | copy));
        b.w = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] >> 17) & 0x7f80u) | copy));
#pragma unroll
        for (int t = 0; t < MT; ++t)
          acc[t] = Mv<T>::run(__builtin_bit_cast(V8, st.x[t][i]), __builtin_bit_cast(V8, b), acc[t]);
      }
      const bool ok = 2 * s + (q >> 1) < KB;
      const float sc = ok ? mv_scale(code2[st.am], st.a2, off) : 0.f;
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) tot[t][r] = fmaf(sc, acc[t][r], tot[t][r]);
    };
    for (int s = s0; s < s1; s += 2) {
      comp(st[0], s);
      if (s + 2 < s1) load(st[0], s + 2);
      if (s + 1 < s1) {
        comp(st[1], s + 1);
        if (s + 3 < s1) load(st[1], s + 3);
      }
    }
    // the two blocks' sums: lanes 0 .. 31 get x rows 4 q + r of their W row
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) tot[t][r] += __shfl_xor(tot[t][r], 32);
    auto store = [&](int m, int n, float v) {
      if (m >= a.M || n >= w.N) return;
      if (w.bias != nullptr) v += (float)static_cast<const T*>(w.bias)[n];
      static_cast<T*>(a.y)[(int64_t)m * a.ldy + w.col0 + n] = (T)v;
    };
    if constexpr (KS == 1) {
      if (lane < 32)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) store(8 * t + 4 * q + r, row, tot[t][r]);
    } else {
      if (lane < 32)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) red[buf][wave][8 * t + 4 * q + r][lq] = tot[t][r];
      __syncthreads();
      for (int i = tid; i < TPB * MT * 128; i += kMvThreads) {
        const int n = i & 15, m = i / 16 % (MT * 8), tile = i / (MT * 128);
        float v = red[buf][tile * KS][m][n];
#pragma unroll
        for (int j = 1; j < KS; ++j) v += red[buf][tile * KS + j][m][n];
        store(m, ((grp - w.group0) * TPB + tile) * 16 + n, v);
      }
      buf ^= 1;  // the next group's barrier comes before this buffer is written again
    }
  }
}

// Any K and any alignment of the packed bytes: a wavefront per row of W, an element at a time.
template <typename T>
__global__ __launch_bounds__(256) void k_nf4_matvec_any(const Nf4MvArgs a) {
  const int lane = threadIdx.x & 63;
  int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  int wi = 0;
  while (wi < a.n && r >= a.w[wi].N) r -= a.w[wi++].N;
  if (wi == a.n) return;
  const Nf4MvWeight& w = a.w[wi];
  const float off = *w.offset;
  float sum[kNf4MvRows];
#pragma unroll
  for (int m = 0; m < kNf4MvRows; ++m) sum[m] = 0.f;
  for (int k = lane; k < a.K; k += 64) {
    const int64_t e = r * a.K + k, f = e >> 6;
    const uint32_t byte = static_cast<const uint8_t*>(w.packed)[e >> 1];
    const float v = w.nf4[(e & 1) ? (byte & 15u) : (byte >> 4)] *
                    mv_scale(w.code2[w.absmax[f]], w.absmax2[f >> 8], off);
#pragma unroll
    for (int m = 0; m < kNf4MvRows; ++m)
      if (m < a.M)
        sum[m] = fmaf((float)static_cast<const T*>(a.x)[(int64_t)m * a.ldx + k], v, sum[m]);
  }
#pragma unroll
  for (int m = 0; m < kNf4MvRows; ++m) {
    if (m >= a.M) break;
    float v = sum[m];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if (lane != 0) continue;
    if (w.bias != nullptr) v += (float)static_cast<const T*>(w.bias)[r];
    static_cast<T*>(a.y)[(int64_t)m * a.ldy + w.col0 + r] = (T)v;
  }
}

template <typename T, int MT, int KS>
void run(Nf4MvArgs& a, hipStream_t s) {
  constexpr int TPB = kMvWaves / KS;
  a.groups = 0;
  for (int i = 0; i < a.n; ++i) {
    a.w[i].group0 = a.groups;
    a.groups += ((a.w[i].N + 15) / 16 + TPB - 1) / TPB;  // a group's tiles are of one weight
  }
  const int blocks = a.groups < 512 ? a.groups : 512;
  hipLaunchKernelGGL((k_nf4_matvec<T, MT, KS>), dim3((unsigned)blocks), dim3(kMvThreads), 0, s, a);
}

template <typename T, int MT>
void run_ks(Nf4MvArgs& a, int64_t tiles, hipStream_t s) {
  int ks = 1;
  while (ks < 8 && tiles * ks < 2048) ks *= 2;
  if (ks == 1) return run<T, MT, 1>(a, s);
  if (ks == 2) return run<T, MT, 2>(a, s);
  if (ks == 4) return run<T, MT, 4>(a, s);
  run<T, MT, 8>(a, s);
}

template <typename T>
void run_t(Nf4MvArgs& a, hipStream_t s) {
  int64_t rows = 0, tiles = 0;
  bool whole = a.K % 64 == 0 && a.ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  for (int i = 0; i < a.n; ++i) {
    rows += a.w[i].N;
    tiles += (a.w[i].N + 15) / 16;
    whole = whole && (reinterpret_cast<uintptr_t>(a.w[i].packed) & 15) == 0;
  }
  if (!whole)
    hipLaunchKernelGGL((k_nf4_matvec_any<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
  else if (a.M <= 8)
    run_ks<T, 1>(a, tiles, s);
  else
    run_ks<T, 2>(a, tiles, s);
}

}  // namespace

hipError_t launch_nf4_matvec(const Nf4MvArgs& args, int dt, hipStream_t s, bool* sup) {
  Nf4MvArgs a = args;
  *sup = dt == 1 || dt == 2;
  if (dt == 1) run_t<_Float16>(a, s);
  if (dt == 2) run_t<__bf16>(a, s);
  return *sup ? hipGetLastError() : hipErrorInvalidValue;
}

}  // namespace esep
