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
// A block takes a run of tiles of 16 W rows; the tiles' 128-k steps, laid end to end, are cut into equal runs,
// one to each of its 16 wavefronts, which streams its run four steps ahead with no barrier; parts of a tile
// meet in LDS at the end and are added in the wavefronts' order. x lies in LDS where it fits.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"
#include "nf4.hpp"

namespace esep {
namespace {

constexpr int kMvThreads = 1024, kMvWaves = 16;
constexpr int kMvTiles = 16;  // tiles of a block at most

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

// What a wavefront needs of 128 k of W: 16 bytes of its lane's row and its block's scale.
struct MvStage {
  uint4 w;
  uint8_t am;
  float a2;
};

// x in LDS (XL): rows of K + 8 elements, so that the 8 rows that a read touches lie in different banks.
constexpr int kMvXBytes = 80 * 1024;
inline bool mv_x_fits(int M, int K) { return (int64_t)M * (K + 8) * 2 <= kMvXBytes; }

template <typename T, int MT, bool XL>
__global__ __launch_bounds__(kMvThreads, 4) void k_nf4_matvec(const Nf4MvArgs a) {
  using V8 = typename Mv<T>::v8;
  __shared__ __align__(16) uint32_t tab[256 * 32];
  __shared__ float code2[256];
  __shared__ float red[kMvWaves + kMvTiles - 1][MT * 8][16];  // a wavefront's part of a tile: [both numbers' sum]
  __shared__ __align__(16) char xs[XL ? kMvXBytes : 16];      // [M][K + 8]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 15, q = lane >> 4;
  const int KB = a.K / 64, steps = (KB + 1) / 2;
  int wi = 0;
  while (wi + 1 < a.n && (int)blockIdx.x >= a.w[wi + 1].block0) ++wi;
  const Nf4MvWeight& w = a.w[wi];
  const int all = (w.N + 15) / 16, tile0 = ((int)blockIdx.x - w.block0) * a.per_block;
  const int tiles = all - tile0 < a.per_block ? all - tile0 : a.per_block;
  const int total = tiles * steps;
  const int waves = total < kMvWaves ? total : kMvWaves;  // each has a step or more
  const int u0 = wave < waves ? wave * total / waves : 0;
  const int u1 = wave < waves ? (wave + 1) * total / waves : 0;

  // the load cursor: step ls of tile lt, this lane's W row in it
  const char* wp;
  const uint8_t* ap;
  int64_t f0;
  auto seek = [&](int lt) {
    const int row = (tile0 + lt) * 16 + lq, rc = row < w.N ? row : w.N - 1;
    wp = static_cast<const char*>(w.packed) + (int64_t)rc * KB * 32 + 16 * q;
    f0 = (int64_t)rc * KB + (lane >> 5);
    ap = w.absmax + f0;
  };
  int lt = u0 / steps, ls = u0 % steps, lu = u0;
  seek(lt);
  auto load = [&](MvStage& st) {
    if (lu >= u1) return;
    const bool ok = 2 * ls + (q >> 1) < KB;
    st.w = ok ? *reinterpret_cast<const uint4*>(wp + 64 * ls) : make_uint4(0, 0, 0, 0);
    st.am = ok ? ap[2 * ls] : 0;
    st.a2 = ok ? w.absmax2[(f0 + 2 * ls) >> 8] : 0.f;
    ++lu;
    if (++ls == steps) {
      ls = 0;
      seek(++lt);
    }
  };
  constexpr int DEPTH = 4;
  MvStage st[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(st[d]);

  // the tables and x, while the first bytes of W are on their way
  const float off = *w.offset;
  {
    const float code = w.nf4[lane & 15];
    for (int i = tid; i < 256 * 8; i += kMvThreads) {
      const int e = i / 8;
      const uint32_t p = mv_pair<T>(__shfl(code, e >> 4), __shfl(code, e & 15));
      reinterpret_cast<uint4*>(tab)[i] = make_uint4(p, p, p, p);
    }
    if (tid < 256) code2[tid] = w.code2[tid];
    if constexpr (XL) {
      const int chunks = a.K / 8;
      for (int i = tid; i < a.M * chunks; i += kMvThreads) {
        const int m = i / chunks, c = i % chunks;
        *reinterpret_cast<uint4*>(xs + ((int64_t)m * (a.K + 8) + 8 * c) * 2) =
            *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (int64_t)m * a.ldx + 8 * c);
      }
    }
  }
  __syncthreads();

  // x: this lane's row of each 8, against its own block's lanes only
  const bool mine = (q >> 1) == (lq >> 3);
  const char* xp[MT];
  bool have[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = 8 * t + (lq & 7);
    have[t] = mine && m < a.M;
    xp[t] = XL ? xs + ((int64_t)m * (a.K + 8) + 32 * q) * 2
               : reinterpret_cast<const char*>(static_cast<const T*>(a.x) + (int64_t)m * a.ldx + 32 * q);
  }
  const uint32_t copy = 4 * (lane & 31);
  const char* tabb = reinterpret_cast<const char*>(tab);
  f32x4 tot[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) tot[t] = f32x4{};
  int ct = u0 / steps, cs = u0 % steps;  // the compute cursor
  auto comp = [&](const MvStage& st, int u) {
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{};
    const bool ok = 2 * cs + (q >> 1) < KB;
    const uint32_t wd[4] = {st.w.x, st.w.y, st.w.z, st.w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint4 b;
      b.x = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] << 7) & 0x7f80u) | copy));
      b.y = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] >> 1) & 0x7f80u) | copy));
      b.z = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] >> 9) & 0x7f80u) | copy));
      b.w = *reinterpret_cast<const uint32_t*>(tabb + (((wd[i] >> 17) & 0x7f80u) | copy));
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (have[t] && ok) x = *reinterpret_cast<const uint4*>(xp[t] + 256 * cs + 16 * i);
        acc[t] = Mv<T>::run(__builtin_bit_cast(V8, x), __builtin_bit_cast(V8, b), acc[t]);
      }
    }
    const float sc = ok ? mv_scale(code2[st.am], st.a2, off) : 0.f;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) tot[t][r] = fmaf(sc, acc[t][r], tot[t][r]);
    if (++cs == steps || u + 1 == u1) {
      // the two blocks' sums: lanes 0 .. 31 hold x rows 4 q + r of their W row
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = tot[t][r] + __shfl_xor(tot[t][r], 32);
          if (lane < 32) red[wave + ct][8 * t + 4 * q + r][lq] = v;
          tot[t][r] = 0.f;
        }
      cs = 0;
      ++ct;
    }
  };
  for (int u = u0; u < u1; u += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (u + d < u1) {
        comp(st[d], u + d);
        load(st[d]);
      }
    }
  }
  __syncthreads();
  // a tile's parts, one of each wavefront that walked some of it, in their order
  for (int i = tid; i < tiles * MT * 128; i += kMvThreads) {
    const int c = i & 15, m = i / 16 % (MT * 8), t = i / (MT * 128);
    const int n = (tile0 + t) * 16 + c;
    if (m >= a.M || n >= w.N) continue;
    const int first = ((t * steps + 1) * waves - 1) / total;
    const int last = ((t + 1) * steps * waves - 1) / total;
    float v = red[first + t][m][c];
    for (int j = first + 1; j <= last; ++j) v += red[j + t][m][c];
    if (w.bias != nullptr) v += (float)static_cast<const T*>(w.bias)[n];
    static_cast<T*>(a.y)[(int64_t)m * a.ldy + w.col0 + n] = (T)v;
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

template <typename T, int MT, bool XL>
hipError_t run(Nf4MvArgs& a, hipStream_t s) {
  // the fewest tiles to a block that one block to a CU holds, up to kMvTiles
  int blocks = 0;
  for (a.per_block = 1;; ++a.per_block) {
    blocks = 0;
    for (int i = 0; i < a.n; ++i) {
      a.w[i].block0 = blocks;
      blocks += ((a.w[i].N + 15) / 16 + a.per_block - 1) / a.per_block;
    }
    if (blocks <= 256 || a.per_block == kMvTiles) break;
  }
  hipLaunchKernelGGL((k_nf4_matvec<T, MT, XL>), dim3((unsigned)blocks), dim3(kMvThreads), 0, s, a);
  return hipGetLastError();
}

template <typename T, int MT>
hipError_t run_x(Nf4MvArgs& a, hipStream_t s) {
  return mv_x_fits(a.M, a.K) ? run<T, MT, true>(a, s) : run<T, MT, false>(a, s);
}

template <typename T>
hipError_t run_t(Nf4MvArgs& a, hipStream_t s) {
  int64_t rows = 0;
  bool whole = a.K % 64 == 0 && a.ldx % 8 == 0 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  for (int i = 0; i < a.n; ++i) {
    rows += a.w[i].N;
    whole = whole && (reinterpret_cast<uintptr_t>(a.w[i].packed) & 15) == 0;
  }
  if (whole) return a.M <= 8 ? run_x<T, 1>(a, s) : run_x<T, 2>(a, s);
  hipLaunchKernelGGL((k_nf4_matvec_any<T>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_nf4_matvec(const Nf4MvArgs& args, int dt, hipStream_t s, bool* sup) {
  Nf4MvArgs a = args;
  *sup = dt == 1 || dt == 2;
  if (dt == 1) return run_t<_Float16>(a, s);
  if (dt == 2) return run_t<__bf16>(a, s);
  return hipErrorInvalidValue;
}

}  // namespace esep
