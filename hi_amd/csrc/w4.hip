// Products with 4-bit weights and group scales, for the few rows of a decode
// step (the reference's models are quantised in groups; its 4-bit row
// products start at crates/hi-cuda/src/kernels.cu:8658).
//
//     w[n][k] = (q[n][k] - z[n][k / G]) * s[n][k / G],   q in 0 .. 15
//     y[m][n] = sum_k x[m][k] * w[n][k] + bias[n]
//
// The weights meet the matrix cores as 16 + q in bf16, which is exact (16 has
// exponent 4, so the upper four mantissa bits count in ones) and costs a shift
// and an and-or for two weights.  A group's product with the rows, d = sum x
// (16 + q), and the rows' sums over the group, e = sum x (a product with ones,
// in the same layout), give
//     y += s * (d - (16 + z) * e)
// in f32: the weights are never rounded.  (An offset of 128, which needs no
// shift for the first pair, would lose three more bits to the difference.)
//
// hi_rocm_w4_pack lays the weights out once: blocks of 16 outputs x 128 inputs
// in the order in which the lanes of a wave hold them, so a wave reads 1 KB
// of contiguous memory a block; the blocks of 16 outputs follow each other
// along k.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "hi_rocm.h"
#include "sampler_internal.h"

namespace hi_rocm {
hipError_t ensure_lds(const void* fn, size_t bytes);  // sampler_chunked.hip

namespace {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w4_u32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4Block = 128;   // inputs of a block
constexpr int kW4Waves = 8;     // waves of a workgroup, splitting k

struct W4Layout {
  int64_t n_tiles, k_blocks;
  size_t scales, zeros, total;
};
W4Layout w4_layout(int n, int k, int group, int scale_dtype, bool zeros) {
  auto align = [](size_t x) { return (x + 255) & ~(size_t)255; };
  W4Layout L;
  L.n_tiles = ((int64_t)n + 15) / 16;
  L.k_blocks = ((int64_t)k + kW4Block - 1) / kW4Block;
  const size_t blocks = (size_t)L.n_tiles * L.k_blocks;
  const size_t per = 16 * (kW4Block / group) * (scale_dtype == HI_ROCM_DTYPE_BF16 ? 2 : 4);
  L.scales = align(blocks * 1024);
  L.zeros = L.scales + align(blocks * per);
  L.total = zeros ? L.zeros + align(blocks * per) : L.zeros;
  return L;
}

// Lane (g, r) = 16 g + r of a block holds output r's inputs 32 i + 8 g .. + 7
// in word i; input 2 p of the eight in nibble p, input 2 p + 1 in nibble p + 4,
// so one shift and one mask give a pair.
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* q, int n, int k, int64_t k_blocks,
                                                      int64_t words, uint32_t* out) {
  const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (w >= words) return;
  const int64_t block = w >> 8;
  const int i = (int)(w & 3), lane = (int)(w >> 2) & 63, r = lane & 15, g = lane >> 4;
  const int64_t row = block / k_blocks * 16 + r, k0 = block % k_blocks * kW4Block + 32 * i + 8 * g;
  uint32_t v = 0u;
  if (row < n && k0 < k) {
    const uint8_t* p = q + row * (k / 2) + k0 / 2;
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t b = p[j];
      v |= (b & 15u) << (4 * j) | (b >> 4) << (4 * j + 16);
    }
  }
  out[w] = v;
}

// Scales (or zeros): [n][k / G] to [block][16][128 / G].  Places past n or k
// hold 0: a scale of 0 drops their products.
template <typename T>
__global__ void __launch_bounds__(256) w4_pack_scales_kernel(const T* in, int n, int groups, int gpb, int64_t k_blocks,
                                                             int64_t count, T* out) {
  const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (w >= count) return;
  const int64_t block = w / (16 * gpb);
  const int j = (int)(w % gpb), r = (int)(w / gpb) & 15;
  const int64_t row = block / k_blocks * 16 + r, grp = block % k_blocks * gpb + j;
  out[w] = row < n && grp < groups ? in[row * groups + grp] : (T)0.f;
}

struct W4Args {
  const __bf16* x;        // [rows][x_stride]
  int64_t x_stride;
  const uint32_t* q;      // packed blocks
  const void* scales;
  const void* zeros;      // or null: 8
  const float* bias;      // or null
  void* out;
  int64_t out_stride;
  int rows, n, k, out_bf16;
  int n_tiles, k_blocks;
};

// The eight weights of a word as 16 + q in bf16: a shift and an and-or for two.
// (`mask` and `sixteens` are 0x00780078 and 0x41804180, a scalar and a vector
// register to the compiler: as literals neither would fit the and-or.)
__device__ __forceinline__ w4_bf16x8 w4_unpack(uint32_t w, uint32_t mask, uint32_t sixteens) {
  const w4_u32x4 v = {((w << 3) & mask) | sixteens, ((w >> 1) & mask) | sixteens, ((w >> 5) & mask) | sixteens,
                      ((w >> 9) & mask) | sixteens};
  return __builtin_bit_cast(w4_bf16x8, v);
}

// The scales (or zeros) that a lane needs of a block: those of its output, as
// one load.
template <typename ST, int GPB>
struct W4Scales {
  typedef ST vec __attribute__((ext_vector_type(GPB)));
  vec v;
  __device__ __forceinline__ void load(const void* p, int64_t block, int r) {
    v = *reinterpret_cast<const vec*>((const ST*)p + (block * 16 + r) * GPB);
  }
  __device__ __forceinline__ float get(int j) const { return (float)v[j]; }
};
template <typename ST>
struct W4Scales<ST, 1> {
  ST v;
  __device__ __forceinline__ void load(const void* p, int64_t block, int r) { v = ((const ST*)p)[block * 16 + r]; }
  __device__ __forceinline__ float get(int) const { return (float)v; }
};

// A workgroup of eight waves takes groups of T tiles of 16 outputs, 16 MT rows
// of x.  Its waves split k: in a pass each owns BPW blocks, whose part of x it
// holds in registers while the weights of tile after tile stream past, R steps
// (a step: a wave's BPW blocks of one tile) ahead, from group to group without
// a pause.  So a weight is read once, nothing but weights is read in the loop
// (x again in every pass, where k is longer than one), and the waves meet once
// a group to add their sums, in wave order, through LDS.
//
// A group's e does not depend on the output: each wave makes it once a pass (a
// product with ones) and keeps -24 e (-e with zeros) in LDS.  What goes into the
// sum, s (d - (16 + z) e), follows one group behind, while the next group's
// product runs.  (Products that start from -24 e would save an addition, but
// weights of 0 would then not give 0.)
// MQ = 1: one row of x; of the four rows a lane's results hold only the first
// is kept (4096 x 65536: 26.4 us, with all four 28.2).
//
// What bounds it: the weights' bytes for a row (4096 x 151936 in groups of 32,
// 350 MB with the scales: 62 us, 5.6 TB/s), the latency of the loads and of the
// two barriers for small weights (1184 x 1000: 6.6 us), and for more rows x,
// which every CU reads from the L2s: 32 rows, 4096 x 16384 with zeros in groups
// of 128, 35 MB of weights: 16.7 us, of which the 64 MB of x in all take 7 (16
// rows: 3.5 of 12).
// MFMA 16x16x32 bf16 (lane l = 16 g + r): A row r, elements 8 g .. 8 g + 7;
// B column r, the same elements; D rows 4 g .. 4 g + 3 of column r.  Rows past
// the last repeat it and are dropped.
template <int MT, int MQ, int T, int BPW, int R, int G, bool ZEROS, typename ST>
__global__ void __launch_bounds__(64 * kW4Waves) w4_linear_kernel(W4Args a) {
  constexpr int GPB = kW4Block / G, CH = G / 32;  // groups a block, MFMAs a group
  constexpr int PART = kW4Waves * T * MT * 64;    // values of the waves' sums
  constexpr bool TWO = MT == 1;                   // two buffers of them
  static_assert(T == 1 || R == T, "a step's tile is its ring slot");
  extern __shared__ __align__(16) float w4_lds[];
  typedef float sums __attribute__((ext_vector_type(MQ)));
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int groups = (a.n_tiles + T - 1) / T;
  const int passes = (a.k_blocks + kW4Waves * BPW - 1) / (kW4Waves * BPW);
  const int m0 = blockIdx.y * (16 * MT);
  // this wave's e: [block][group][row tile][g] of four rows
  w4_f32x4* ex = reinterpret_cast<w4_f32x4*>(w4_lds + (TWO ? 2 : 1) * PART * MQ) + wid * (BPW * GPB * MT * 4) + g;
  const __bf16* xr[MT];
  #pragma unroll
  for (int m = 0; m < MT; ++m) xr[m] = a.x + (int64_t)min(m0 + 16 * m + r, a.rows - 1) * a.x_stride + 8 * g;
  uint32_t mask = 0x00780078u, sixteens = 0x41804180u;
  asm volatile("" : "+s"(mask), "+v"(sixteens));

  w4_u32x4 wv[R][BPW];
  W4Scales<ST, GPB> sv[R][BPW], zv[R][BPW];
  // the step to load next: tile t of a group, in a pass
  int lg = blockIdx.x, lp = 0, lt = 0;
  auto load = [&](int slot) {
    const int nt = min(lg * T + lt, a.n_tiles - 1);  // (past the last step: loads that nothing uses)
    #pragma unroll
    for (int i = 0; i < BPW; ++i) {
      const int64_t block = (int64_t)nt * a.k_blocks + min((lp * kW4Waves + wid) * BPW + i, a.k_blocks - 1);
      wv[slot][i] = *reinterpret_cast<const w4_u32x4*>(a.q + block * 256 + lane * 4);
      sv[slot][i].load(a.scales, block, r);
      if (ZEROS) zv[slot][i].load(a.zeros, block, r);
    }
    if (++lt == T) {
      lt = 0;
      if (++lp == passes) {
        lp = 0;
        lg += gridDim.x;
      }
    }
  };
  w4_bf16x8 xf[BPW][4][MT];
  auto load_x = [&](int pass) {
    #pragma unroll
    for (int i = 0; i < BPW; ++i) {
      #pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = ((pass * kW4Waves + wid) * BPW + i) * kW4Block + 32 * j;
        // (in steps of 32, k is inside or outside as a whole; every load is made)
        const uint32_t in = k < a.k ? ~0u : 0u;
        #pragma unroll
        for (int m = 0; m < MT; ++m) {
          const w4_u32x4 v = *reinterpret_cast<const w4_u32x4*>(xr[m] + min(k, a.k - 32));
          xf[i][j][m] = __builtin_bit_cast(w4_bf16x8, v & in);
        }
      }
    }
    w4_bf16x8 ones;
    #pragma unroll
    for (int i = 0; i < 8; ++i) ones[i] = (__bf16)1.0f;
    #pragma unroll
    for (int i = 0; i < BPW; ++i) {
      #pragma unroll
      for (int j = 0; j < GPB; ++j) {
        #pragma unroll
        for (int m = 0; m < MT; ++m) {
          w4_f32x4 e = {0.f, 0.f, 0.f, 0.f};
          #pragma unroll
          for (int c = j * CH; c < (j + 1) * CH; ++c)
            e = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i][c][m], ones, e, 0, 0, 0);
          if (r == 0) ex[((i * GPB + j) * MT + m) * 4] = ZEROS ? -e : -24.f * e;
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  };
  sums acc[T][MT];
  auto clear = [&]() {
    #pragma unroll
    for (int t = 0; t < T; ++t)
      #pragma unroll
      for (int m = 0; m < MT; ++m)
        #pragma unroll
        for (int q = 0; q < MQ; ++q) acc[t][m][q] = 0.f;
  };
  auto multiply = [&](int slot, int t) {
    w4_f32x4 d[2][MT], e[2][MT];
    float s[2], z[2];
    auto add = [&](int p) {
      #pragma unroll
      for (int m = 0; m < MT; ++m)
        #pragma unroll
        for (int q = 0; q < MQ; ++q) {
          // (group after group: all at once would not fit the registers)
          const float w = ZEROS ? fmaf(z[p], e[p][m][q], d[p][m][q]) : d[p][m][q] + e[p][m][q];
          float v = fmaf(s[p], w, acc[t][m][q]);
          asm volatile("" : "+v"(v));
          acc[t][m][q] = v;
        }
    };
    #pragma unroll
    for (int i = 0; i < BPW; ++i) {
      asm volatile("" : "+v"(wv[slot][i]));
      #pragma unroll
      for (int j = 0; j < GPB; ++j) {
        const int p = (i * GPB + j) & 1;
        s[p] = sv[slot][i].get(j);
        if (ZEROS) z[p] = 16.f + zv[slot][i].get(j);
        #pragma unroll
        for (int m = 0; m < MT; ++m) {
          e[p][m] = ex[((i * GPB + j) * MT + m) * 4];
          d[p][m] = w4_f32x4{0.f, 0.f, 0.f, 0.f};
        }
        #pragma unroll
        for (int c = j * CH; c < (j + 1) * CH; ++c) {
          const w4_bf16x8 b = w4_unpack(wv[slot][i][c], mask, sixteens);
          #pragma unroll
          for (int m = 0; m < MT; ++m)
            d[p][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xf[i][c][m], b, d[p][m], 0, 0, 0);
        }
        if (i + j > 0) add(p ^ 1);
      }
    }
    add((BPW * GPB - 1) & 1);
  };
  int buffer = 0;
  auto finish = [&](int grp) {
    sums* part = reinterpret_cast<sums*>(w4_lds) + buffer * PART;
    #pragma unroll
    for (int t = 0; t < T; ++t)
      #pragma unroll
      for (int m = 0; m < MT; ++m) part[((wid * T + t) * MT + m) * 64 + lane] = acc[t][m];
    __syncthreads();
    for (int i = threadIdx.x; i < T * MT * 64; i += 64 * kW4Waves) {
      const int l = i & 63, m = i / 64 % MT, t = i / 64 / MT;
      const int n = (grp * T + t) * 16 + (l & 15), row = m0 + 16 * m + 4 * (l >> 4);
      if (n >= a.n || row >= a.rows) continue;
      sums y = part[i];
      #pragma unroll
      for (int w = 1; w < kW4Waves; ++w) y += part[w * T * MT * 64 + i];
      const float bias = a.bias ? a.bias[n] : 0.f;
      #pragma unroll
      for (int q = 0; q < MQ; ++q) {
        if (row + q >= a.rows) break;
        const float v = a.bias ? y[q] + bias : y[q];
        const int64_t at = (int64_t)(row + q) * a.out_stride + n;
        if (a.out_bf16) ((__bf16*)a.out)[at] = (__bf16)v;
        else ((float*)a.out)[at] = v;
      }
    }
    // (with two buffers the next group's barrier keeps the one after it off this one)
    if (TWO) buffer ^= 1;
    else __syncthreads();
  };

  #pragma unroll
  for (int s = 0; s < R; ++s) load(s);
  load_x(0);
  clear();
  int grp = blockIdx.x, pass = 0;
  while (grp < groups) {
    #pragma unroll
    for (int s = 0; s < R; ++s) {
      const int t = T == 1 ? 0 : s;
      if (grp < groups) {
        if (passes > 1 && t == 0) load_x(pass);
        multiply(s, t);
        load(s);
        if (t == T - 1 && ++pass == passes) {
          finish(grp);
          clear();
          pass = 0;
          grp += gridDim.x;
        }
      }
    }
  }
}

template <int MT, int MQ, int T, int BPW, int R, int G, bool ZEROS, typename ST>
hipError_t launch_w4(const W4Args& a, hipStream_t st) {
  const size_t bytes = (size_t)kW4Waves * sizeof(float) *
                       ((MT == 1 ? 2 : 1) * T * MT * 64 * MQ + BPW * (kW4Block / G) * MT * 16);
  auto* kernel = w4_linear_kernel<MT, MQ, T, BPW, R, G, ZEROS, ST>;
  const hipError_t e = ensure_lds((const void*)kernel, bytes);
  if (e != hipSuccess) return e;
  // one workgroup a CU stays and takes every 256th group
  const int groups = (a.n_tiles + T - 1) / T;
  const dim3 grid((unsigned)std::min(groups, 256), (unsigned)((a.rows + 16 * MT - 1) / (16 * MT)));
  hipLaunchKernelGGL(kernel, grid, dim3(64 * kW4Waves), bytes, st, a);
  return hipGetLastError();
}
// T and BPW.  Up to 16 blocks of k one pass holds all of x with BPW = 1 or 2;
// then T = 1 while that is at most two workgroups a CU, else T = 4.  Longer k
// takes T = 1 (in passes of 8 blocks) while that is at most one workgroup a CU,
// else T = 2 with BPW = 4, a pass of up to 32 blocks, and beyond those T = 4
// where T = 2 would be more than one workgroup a CU.  Whole calls, us (bf16
// scales, groups of 32, k x n):
//   1 row, 1024 x 4096: T = 1 3.2, 4 4.1; 1024 x 16384: 4.5 and 4.2;
//     2048 x 8192: 4.7 and 5.7; 2048 x 16384: 6.0 and 6.3; 2048 x 65536: 16.7 and 16.4
//   16 rows, 4096 x 4096: T = 1 8.0, 2 9.0, 4 12.7; 4096 x 16384: 18.3, 13.1, 15.0;
//     1 row, 8192 x 16384: 29.2, 21.4, 18.5; 8192 x 8192: 15.2, 13.5, 16.9
// MT = 2 where MT = 1 would be more than one workgroup a CU: 32 rows, 4096 x
// 65536: 45.0, with MT = 1 59.3; 64 rows, 2048 x 8192: 10.7 and 12.1; but 32 rows,
// 4096 x 4096 (256 workgroups with MT = 1): 14.4 and 9.2.
// (MT = 4 read x too often to gain: 64 rows, 4096 x 65536 110, with MT = 2 86.)
// With f32 scales and zeros for groups of 32, MT = 2 and T = 2 are far from
// fitting the registers: 32 rows, 4096 x 65536: 108, with T = 4 69.  Three other
// types spill 8 to 11 registers there and still win or lose little (32 rows, 4096
// x 65536 with T = 2 and 4, then 4096 x 16384): groups of 32 with bf16 scales and
// zeros 59 and 69, 23.6 and 22.2; with f32 scales 52 and 65, 21.8 and 21.7; of 64
// with f32 scales and zeros 48 and 62, 20.3 and 20.6.
// Beyond 64 rows the weights are unpacked again for every 32 of them: 4096 x
// 14336, 128, 512 and 2,048 rows: 55, 210 and 825 (a bf16 library product of
// unpacked weights 25, 55 and 164).
template <int G, bool ZEROS, typename ST>
hipError_t launch_w4_rows(const W4Args& a, hipStream_t st) {
  const int64_t row_tiles = (a.rows + 15) / 16;
  auto wgs = [&](int t) { return (a.n_tiles + t - 1) / t * row_tiles; };
  const bool shrt = a.k_blocks <= 16;
  const int t = wgs(1) <= (shrt ? 512 : 256) ? 1 : shrt ? 4 : a.k_blocks <= 32 || wgs(2) <= 256 ? 2 : 4;
  const bool one = a.k_blocks <= 8;
  if (a.rows == 1) {
    if (t == 1) return one || !shrt ? launch_w4<1, 1, 1, 1, 3, G, ZEROS, ST>(a, st) : launch_w4<1, 1, 1, 2, 3, G, ZEROS, ST>(a, st);
    if (t == 2) return launch_w4<1, 1, 2, 4, 2, G, ZEROS, ST>(a, st);
    return one ? launch_w4<1, 1, 4, 1, 4, G, ZEROS, ST>(a, st) : launch_w4<1, 1, 4, 2, 4, G, ZEROS, ST>(a, st);
  }
  if (t == 1)
    return one || !shrt ? launch_w4<1, 4, 1, 1, 3, G, ZEROS, ST>(a, st) : launch_w4<1, 4, 1, 2, 3, G, ZEROS, ST>(a, st);
  if (row_tiles == 1 || wgs(t) <= 256) {
    if (t == 2) return launch_w4<1, 4, 2, 4, 2, G, ZEROS, ST>(a, st);
    return one ? launch_w4<1, 4, 4, 1, 4, G, ZEROS, ST>(a, st) : launch_w4<1, 4, 4, 2, 4, G, ZEROS, ST>(a, st);
  }
  if constexpr (G > 32 || !ZEROS || sizeof(ST) == 2)
    if (t == 2) return launch_w4<2, 4, 2, 4, 2, G, ZEROS, ST>(a, st);
  return one ? launch_w4<2, 4, 4, 1, 4, G, ZEROS, ST>(a, st) : launch_w4<2, 4, 4, 2, 4, G, ZEROS, ST>(a, st);
}
template <int G, typename ST>
hipError_t launch_w4_zeros(const W4Args& a, hipStream_t st) {
  return a.zeros ? launch_w4_rows<G, true, ST>(a, st) : launch_w4_rows<G, false, ST>(a, st);
}
template <typename ST>
hipError_t launch_w4_group(const W4Args& a, int group, hipStream_t st) {
  if (group == 32) return launch_w4_zeros<32, ST>(a, st);
  if (group == 64) return launch_w4_zeros<64, ST>(a, st);
  return launch_w4_zeros<128, ST>(a, st);
}

// Sizes and types of a packed weight: HI_ROCM_OK, or a status with a message.
int w4_check(int n, int k, int group, int scale_dtype, const char* what_args, const char* what_sizes) {
  if (n <= 0 || k <= 0 || group <= 0 || (scale_dtype != HI_ROCM_DTYPE_F32 && scale_dtype != HI_ROCM_DTYPE_BF16))
    return api_fail(HI_ROCM_ERR_ARGS, what_args);
  if ((group != 32 && group != 64 && group != 128) || k % group != 0 || n > (1 << 24) || k > (1 << 24))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, what_sizes);
  return HI_ROCM_OK;
}

}  // namespace
}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_w4_packed_bytes(int n, int k, int group, int scale_dtype, int has_zeros, size_t* out_bytes) {
  if (out_bytes == nullptr) return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_packed_bytes: invalid arguments");
  const int rc = w4_check(n, k, group, scale_dtype, "hi_rocm_w4_packed_bytes: invalid arguments",
                          "hi_rocm_w4_packed_bytes: needs groups of 32, 64 or 128, k a multiple of them, n and k up to 2^24");
  if (rc != HI_ROCM_OK) return rc;
  *out_bytes = w4_layout(n, k, group, scale_dtype, has_zeros != 0).total;
  return HI_ROCM_OK;
}

int hi_rocm_w4_pack(const void* q, const void* scales, const void* zeros, int scale_dtype, int n, int k, int group,
                    void* packed, size_t packed_bytes, void* stream) {
  if (q == nullptr || scales == nullptr || packed == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_pack: invalid arguments");
  const int rc = w4_check(n, k, group, scale_dtype, "hi_rocm_w4_pack: invalid arguments",
                          "hi_rocm_w4_pack: needs groups of 32, 64 or 128, k a multiple of them, n and k up to 2^24");
  if (rc != HI_ROCM_OK) return rc;
  const W4Layout L = w4_layout(n, k, group, scale_dtype, zeros != nullptr);
  if (packed_bytes < L.total || (uintptr_t)packed % 16 != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_pack: packed buffer too small or not 16-byte aligned");
  if ((uintptr_t)scales % (scale_dtype == HI_ROCM_DTYPE_BF16 ? 2 : 4) != 0 ||
      (uintptr_t)zeros % (scale_dtype == HI_ROCM_DTYPE_BF16 ? 2 : 4) != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_pack: scales not aligned to their type");
  const int64_t blocks = L.n_tiles * L.k_blocks, words = blocks * 256;
  const int gpb = kW4Block / group;
  const int64_t count = blocks * 16 * gpb;
  if (words > UINT32_MAX - 255)  // a thread each
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_w4_pack: more than 2^35 weights");
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(w4_pack_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, st, (const uint8_t*)q, n, k,
                     L.k_blocks, words, (uint32_t*)packed);
  for (int i = 0; i < (zeros ? 2 : 1); ++i) {
    const void* in = i ? zeros : scales;
    char* out = (char*)packed + (i ? L.zeros : L.scales);
    const dim3 grid((unsigned)((count + 255) / 256));
    if (scale_dtype == HI_ROCM_DTYPE_BF16)
      hipLaunchKernelGGL(w4_pack_scales_kernel<__bf16>, grid, dim3(256), 0, st, (const __bf16*)in, n, k / group, gpb,
                         L.k_blocks, count, (__bf16*)out);
    else
      hipLaunchKernelGGL(w4_pack_scales_kernel<float>, grid, dim3(256), 0, st, (const float*)in, n, k / group, gpb,
                         L.k_blocks, count, (float*)out);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "w4 pack launch");
}

int hi_rocm_w4_linear(const void* x, int rows, int64_t x_stride, const void* packed, size_t packed_bytes,
                      int scale_dtype, int has_zeros, int n, int k, int group, const float* bias, void* out,
                      int out_dtype, int64_t out_stride, void* stream) {
  if (x == nullptr || packed == nullptr || out == nullptr || rows <= 0 || x_stride < k || out_stride < n ||
      (out_dtype != HI_ROCM_DTYPE_F32 && out_dtype != HI_ROCM_DTYPE_BF16))
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_linear: invalid arguments");
  const int rc = w4_check(n, k, group, scale_dtype, "hi_rocm_w4_linear: invalid arguments",
                          "hi_rocm_w4_linear: needs groups of 32, 64 or 128, k a multiple of them, n and k up to 2^24");
  if (rc != HI_ROCM_OK) return rc;
  if (rows > 16 * 65535)  // (a grid's second dimension)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_w4_linear: more than 16 * 65535 rows");
  if ((uintptr_t)x % 16 != 0 || x_stride % 8 != 0)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_w4_linear: needs rows of x that start on 16 bytes");
  if ((uintptr_t)out % (out_dtype == HI_ROCM_DTYPE_F32 ? 4 : 2) != 0 || (uintptr_t)bias % 4 != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_linear: out or bias not aligned to its type");
  const W4Layout L = w4_layout(n, k, group, scale_dtype, has_zeros != 0);
  if (packed_bytes < L.total || (uintptr_t)packed % 16 != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_w4_linear: packed buffer too small or not 16-byte aligned");
  W4Args a;
  memset(&a, 0, sizeof(a));
  a.x = (const __bf16*)x;
  a.x_stride = x_stride;
  a.q = (const uint32_t*)packed;
  a.scales = (const char*)packed + L.scales;
  a.zeros = has_zeros ? (const char*)packed + L.zeros : nullptr;
  a.bias = bias;
  a.out = out;
  a.out_stride = out_stride;
  a.rows = rows;
  a.n = n;
  a.k = k;
  a.out_bf16 = out_dtype == HI_ROCM_DTYPE_BF16;
  a.n_tiles = (int)L.n_tiles;
  a.k_blocks = (int)L.k_blocks;
  const hipError_t e = scale_dtype == HI_ROCM_DTYPE_BF16 ? launch_w4_group<__bf16>(a, group, (hipStream_t)stream)
                                                         : launch_w4_group<float>(a, group, (hipStream_t)stream);
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "w4 linear launch");
}

}  // extern "C"
