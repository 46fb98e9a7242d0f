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
// The codes are rounded to x's type, the matrix instructions' operand type, as dequantize_nf4 rounds the whole weight
// to it: by up to 2^-11.6 of a code in fp16 and 2^-8.3 in bf16 (2^-12.5 and 2^-9.5 in the root mean square), the same
// for each of the 16 wherever it stands. Scales, products and sums stay in fp32.
//
// A block takes a run of tiles of 16 W rows; the tiles' 128-k steps, laid end to end, are cut into equal runs,
// one to each of its 16 wavefronts, which streams its run four steps ahead with no barrier; parts of a tile
// meet in LDS at the end and are added in the wavefronts' order. x lies in LDS where it fits.
//
// Kernel trace, one row of x in fp16: 2 x 18944 rows of W of 3584 in 20.6 us (70 MB, 3.4 TB/s; 14.0 is the copy
// rate's time), q / k / v of 1536 in 7.0; 7 rows in bf16, 1536 of 8960 in 11.4 (96 blocks for 256 CUs; a finer
// cut, parts of a tile added across blocks, was not tried). Parts left out in a copy for timing, 20.3 us
// with all: without the table reads 19.2, without the loads of W 16.9, so loads and decode overlap. Slower: six or
// eight steps ahead (21.0, 22.8), x in registers (20.8), loads of 128 bytes of a row (21.0), W past the caches
// (22.4).
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

// A wavefront's loads of one step (128 k): 16 bytes of W a lane, four lanes to the 64 bytes of a row, as memory
// lies; the products want neighbouring lanes in neighbouring rows, which goes through 1 KiB of LDS of the
// wavefront's own. x, where it comes from global memory, likewise: 16 lanes to a row.
template <int XT>
struct MvStage {
  u32x4 w;
  u32x4 x[2 * XT];
};

// x in LDS (XL): rows of whole steps, zeros behind K, and 8 elements more, so that the 8 rows that a
// read touches lie in different banks; before them 64 bytes of zeros that the lanes without a row read.
// Otherwise each wavefront writes its step of x there, in the same form.
constexpr int mv_x_bytes(int MT) { return (MT == 1 ? 95 : 80) * 1024; }  // what a CU's 160 KiB leave
inline __host__ __device__ int mv_x_row(int K) { return 2 * ((K + 127) / 128 * 128 + 8); }
// A block with one tile reads x once, and gains from its copy up to 64 KiB only (8 rows of 5632, 2048 outputs:
// 9.0 us with it, 8.7 without; 10 rows of 3584, 2 x 18944 outputs, ten tiles to a block: 24.9 and 31.4).
inline bool mv_x_fits(int M, int K, int MT, int per_block) {
  return 64 + (int64_t)M * mv_x_row(K) <= (per_block > 1 ? mv_x_bytes(MT) : 64 * 1024);
}

template <typename T, int MT, bool XL>
__global__ __launch_bounds__(kMvThreads, 4) void k_nf4_matvec(const Nf4MvArgs a) {
  using V8 = typename Mv<T>::v8;
  constexpr int XT = XL ? 0 : MT, XW = 8 * MT * 272;  // a wavefront's step of x
  constexpr int DEPTH = XT == 2 ? 2 : 4;              // steps in flight, and scales at a time
  using Stage = MvStage<XT>;
  struct Lds {
    uint32_t tab[256 * 32];  // first: its entries' addresses are then what v_dot4 gives
    float code2[256];
    float red[kMvWaves + kMvTiles - 1][MT * 8][16];  // a wavefront's part of a tile: [both numbers' sum]
    char ws[kMvWaves][1024];                         // a wavefront's step of W
    char xs[XL ? mv_x_bytes(MT) : 64 + kMvWaves * XW];
  };
  __shared__ __align__(16) Lds lds;
  auto& tab = lds.tab;
  auto& code2 = lds.code2;
  auto& red = lds.red;
  auto& ws = lds.ws;
  auto& xs = lds.xs;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lq = lane & 15, q = lane >> 4;
  const int KB = a.K / 64, steps = (KB + 1) / 2;
  int wi = 0;
  while (wi + 1 < a.n && (int)blockIdx.x >= a.w[wi + 1].block0) ++wi;
  const Nf4MvWeight w = a.w[wi];
  const int all = (w.N + 15) / 16, tile0 = ((int)blockIdx.x - w.block0) * a.per_block;
  const int tiles = all - tile0 < a.per_block ? all - tile0 : a.per_block;
  const int total = tiles * steps;
  const int waves = total < kMvWaves ? total : kMvWaves;  // each has a step or more
  const int u0 = wave < waves ? wave * total / waves : 0;
  const int u1 = wave < waves ? (wave + 1) * total / waves : 0;

  // The load cursor: step ls of tile lt. A tile is read through buffer descriptors that end with the weight
  // (and 2 GiB on, past every tile), so that rows and blocks behind its end need no branch: they read 0.
  rsrc_t rw, ra;
  const rsrc_t r2 = make_rsrc(w.absmax2, (uint32_t)(((int64_t)w.N * KB + 255) / 256 * 4));
  const uint32_t vw = (uint32_t)(lane >> 2) * KB * 32 + 16 * (lane & 3);
  const rsrc_t rx = make_rsrc(a.x, XL ? 0 : (uint32_t)(((a.M - 1) * a.ldx + a.K) * 2));
  int64_t f0;
  auto seek = [&](int lt) {
    const int64_t row = (int64_t)(tile0 + lt) * 16, left = (w.N - row) * KB;
    rw = make_rsrc(static_cast<const char*>(w.packed) + row * KB * 32,
                   left < (1 << 26) ? (uint32_t)left * 32 : 0x80000000u);
    ra = make_rsrc(w.absmax + row * KB, left < (1 << 26) ? (uint32_t)left : 1u << 26);
    f0 = row * KB;
  };
  int lt = u0 / steps, ls = u0 % steps, lu = u0;
  seek(lt);
  // The scales of the DEPTH steps from (lt, ls) on, two steps to a register: lane l has row l / 2 % 16 of
  // step l % 2, block l / 32 of it.
  uint32_t am[DEPTH / 2], a2[DEPTH / 2];
  bool in[DEPTH / 2];
  auto load_scales = [&]() {
#pragma unroll
    for (int h = 0; h < DEPTH / 2; ++h) {
      int s = ls + 2 * h + (lane & 1), row = (lane >> 1) & 15;
      if (s >= steps) {  // in the next tile
        const int t = steps < DEPTH ? s / steps : 1;
        s -= t * steps;
        row += 16 * t;
      }
      const int kb = 2 * s + (lane >> 5);
      const uint32_t f = (uint32_t)row * KB + kb;
      in[h] = kb < KB && lu < u1;
      am[h] = __builtin_amdgcn_raw_buffer_load_b8(ra, in[h] ? f : ~0u, 0, 0);
      a2[h] = __builtin_amdgcn_raw_buffer_load_b32(r2, (uint32_t)((f0 + f) >> 8) * 4, 0, 0);
    }
  };
  // (No load stands under a condition: the compiler would wait for all of them at the next use. Past the
  // run's end they go past the buffer's and read nothing.)
  auto load = [&](Stage& st) {
    st.w = __builtin_amdgcn_raw_buffer_load_b128(rw, lu < u1 ? vw : ~0u, 64 * ls, 0);
    if constexpr (!XL) {
#pragma unroll
      for (int t = 0; t < 2 * MT; ++t) {
        const int m = 4 * t + (lane >> 4), k = 128 * ls + 8 * lq;
        // rows and columns behind x read 0
        const bool ok = m < a.M && k < a.K && lu < u1;
        st.x[t] = __builtin_amdgcn_raw_buffer_load_b128(rx, ok ? (uint32_t)(m * a.ldx + k) * 2 : ~0u, 0, 0);
      }
    }
    ++lu;
    if (++ls == steps && lu < u1) {
      ls = 0;
      seek(++lt);
    }
  };
  // What the tables are made of is asked for first: its wait then leaves W's first bytes on their way.
  const float code = w.nf4[lane & 15], code_2 = w.code2[tid & 255];
  load_scales();
  Stage st[DEPTH];
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) load(st[d]);
  const float off = *w.offset;
  // (the bias of the output that this thread adds up first, too)
  const int n0 = (tile0 + tid / (MT * 128)) * 16 + (tid & 15);
  const float bias0 = w.bias != nullptr && n0 < w.N ? (float)static_cast<const T*>(w.bias)[n0] : 0.f;
  for (int i = tid; i < 256 * 8; i += kMvThreads) {
    const int e = i / 8;
    const uint32_t p = mv_pair<T>(__shfl(code, e >> 4), __shfl(code, e & 15));
    reinterpret_cast<uint4*>(tab)[i] = make_uint4(p, p, p, p);
  }
  if (tid < 256) code2[tid] = code_2;
  if (tid < 4) reinterpret_cast<u32x4*>(xs)[tid] = u32x4{0, 0, 0, 0};
  if constexpr (XL) {
    const int chunks = 16 * steps, data = a.K / 8;  // 16-byte pieces of a row
    for (int i = tid; i < a.M * chunks; i += kMvThreads) {
      const int m = i / chunks, c = i % chunks;
      u32x4 v = {0, 0, 0, 0};
      if (c < data)
        v = *reinterpret_cast<const u32x4*>(static_cast<const T*>(a.x) + (int64_t)m * a.ldx + 8 * c);
      *reinterpret_cast<u32x4*>(xs + 64 + m * mv_x_row(a.K) + 16 * c) = v;
    }
  }
  __syncthreads();

  // this lane's place in x: row 8 t + lq % 8, against its own block's lanes only (the others read the
  // zeros), and whether it moves with the steps
  uint32_t xo[MT], xm[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = 8 * t + (lq & 7);
    const bool have = (q >> 1) == (lq >> 3) && m < a.M;
    xo[t] = have ? 64 + (XL ? m * mv_x_row(a.K) : wave * XW + m * 272) + 64 * q : 0;
    xm[t] = XL && have ? ~0u : 0u;
  }
  const uint32_t copy = 4 * (lane & 31);
  const int from_s = 128 * (q >> 1) + 8 * lq;  // 4 times the lane that has this one's scale
  // W's 16-byte pieces in LDS: piece c of row r at 4 r + (c ^ r / 4), so that the 16 rows of a read lie in
  // different banks
  char* to_w = ws[wave] + 64 * (lane >> 2) + 16 * ((lane & 3) ^ (lane >> 4));
  const char* from_w = ws[wave] + 64 * lq + 16 * (q ^ (lq >> 2));
  const char* tabb = reinterpret_cast<const char*>(tab);
  f32x4 tot[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) tot[t] = f32x4{};
  int ct = u0 / steps, cs = u0 % steps;  // the compute cursor
  float sc[DEPTH / 2];
  auto comp = [&](const Stage& st, int u, int d) {
    const float s = __int_as_float(
        __builtin_amdgcn_ds_bpermute(from_s + 4 * (d & 1), __float_as_int(sc[d >> 1])));
    *reinterpret_cast<u32x4*>(to_w) = st.w;
    if constexpr (!XL) {
#pragma unroll
      for (int t = 0; t < 2 * MT; ++t)
        *reinterpret_cast<u32x4*>(xs + 64 + wave * XW + (4 * t + (lane >> 4)) * 272 + 16 * lq) = st.x[t];
    }
    // the wavefront's own LDS operations run in their order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const u32x4 wr = *reinterpret_cast<const u32x4*>(from_w);
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // byte j times 128, one v_dot4, is its entry's place in the table
      u32x4 b;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        b[j] = *reinterpret_cast<const uint32_t*>(
            tabb + __builtin_amdgcn_udot4(wr[i], 128u << (8 * j), copy, false));
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(xs + (xo[t] + ((256u * cs) & xm[t])) + 16 * i);
        acc[t] = Mv<T>::run(__builtin_bit_cast(V8, x), __builtin_bit_cast(V8, b), acc[t]);
      }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) tot[t][r] = fmaf(s, acc[t][r], tot[t][r]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read before the next step is written
    __builtin_amdgcn_wave_barrier();
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
    // a block behind K has a scale of 0: x is 0 there, and what W's next row has does not matter
#pragma unroll
    for (int h = 0; h < DEPTH / 2; ++h)
      sc[h] = in[h] ? mv_scale(code2[am[h] & 255], __uint_as_float(a2[h]), off) : 0.f;
    load_scales();
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (u + d < u1) comp(st[d], u + d, d);
      load(st[d]);
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
    if (w.bias != nullptr) v += i == tid ? bias0 : (float)static_cast<const T*>(w.bias)[n];
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
    float v = sum[m];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if (lane != 0 || m >= a.M) continue;
    if (w.bias != nullptr) v += (float)static_cast<const T*>(w.bias)[r];
    static_cast<T*>(a.y)[(int64_t)m * a.ldy + w.col0 + r] = (T)v;
  }
}

template <typename T, int MT>
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
  if (mv_x_fits(a.M, a.K, MT, a.per_block))
    hipLaunchKernelGGL((k_nf4_matvec<T, MT, true>), dim3((unsigned)blocks), dim3(kMvThreads), 0, s, a);
  else
    hipLaunchKernelGGL((k_nf4_matvec<T, MT, false>), dim3((unsigned)blocks), dim3(kMvThreads), 0, s, a);
  return hipGetLastError();
}

template <typename T>
hipError_t run_t(Nf4MvArgs& a, hipStream_t s) {
  int64_t rows = 0;
  bool whole = a.K % 64 == 0 && a.ldx % 8 == 0 && a.ldx <= 1 << 26 && (reinterpret_cast<uintptr_t>(a.x) & 15) == 0;
  for (int i = 0; i < a.n; ++i) {
    rows += a.w[i].N;
    whole = whole && (reinterpret_cast<uintptr_t>(a.w[i].packed) & 15) == 0;
  }
  if (whole) return a.M <= 8 ? run<T, 1>(a, s) : run<T, 2>(a, s);
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
