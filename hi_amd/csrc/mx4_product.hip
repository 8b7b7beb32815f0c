// Products with microscaled 4-bit weights (mx4.h): linear layers and the
// experts behind the MoE router (moe_experts.hip has the same in bf16, and the
// grouping and combination around both).
//
//     y[i][c] = sum_k Q(x[row(i)])[k] * w[e][c][k] (+ bias[c])
//
// Both operands go to the matrix cores as they lie in memory, 4 bits a value
// with a scale for 32: four times the bf16 rate, and no unpacking.  Q rounds x to
// the same format: beforehand ("rows"), or, for few rows, in registers as it is
// loaded, since a block is one lane's.  Products of two codes are multiples of
// 1/4 up to 36, so a block's sum is exact; the sums over blocks are f32.
//
// MFMA 16x16x128: A row r and B column r in lane 16 g + r, block g; D rows 4 g ..
// + 3 of column r.  Weights are A and places B: a lane ends with four
// neighbouring columns of one place.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "hi_rocm.h"
#include "moe_work.h"
#include "mx4.h"
#include "sampler_internal.h"

namespace hi_rocm {
hipError_t ensure_lds(const void* fn, size_t bytes);  // sampler_chunked.hip
hipError_t mx4_make_rows(const void* x, int dtype, int64_t rows, int k, int64_t x_stride, void* out,
                         hipStream_t st);  // mx4_quantize.hip

namespace {

struct Mx4Args {
  const uint8_t* x;          // bf16 rows, or codes
  int64_t x_stride;          // bytes
  const uint8_t* x_scales;   // with codes
  int64_t x_scale_stride;
  const int32_t* order;      // or null: place i's row is i
  const int32_t* offsets;    // [experts + 1], or null: one expert, all places
  const uint8_t* w;          // packed
  const uint8_t* w_scales;
  const float* bias;         // or null
  void* out;                 // [places][out_stride], or codes
  int64_t out_stride;        // values, or bytes of codes
  uint8_t* out_scales;       // with codes
  int64_t out_scale_stride;
  int x_rows, top_k, places, experts, cols, k, swiglu, out_dtype;
  int tiles, steps, quads;   // of an expert's packed weight
  int out_vec;               // rows of out start on 16 bytes
  int past;                  // results are stored past the caches (mx4_past)
};

// This workgroup's tile of BM places and block of columns.
constexpr int kMx4Rows = 4;
template <int BM>
__device__ __forceinline__ bool mx4_work(const Mx4Args& a, int blocks, MoeWork& wk) {
  if (a.offsets != nullptr) return moe_work<BM>(a, blocks, wk);
  const int nt = (a.places + BM - 1) / BM;
  const int64_t total = (int64_t)nt * blocks, per = (total + kXcds - 1) / kXcds;
  const int64_t slot = blockIdx.x / kXcds, w = blockIdx.x % kXcds * per + slot;
  if (slot >= per || w >= total) return false;
  // One expert: up to kMx4Rows tiles of places by all blocks, then the next tiles.
  // What an XCD's CUs run at a time is then some tiles by some blocks, and its L2
  // serves each of them more than once.
  const int64_t group = w / ((int64_t)kMx4Rows * blocks);
  const int first = (int)group * kMx4Rows, rows = min(nt - first, kMx4Rows);
  const int local = (int)(w - group * kMx4Rows * blocks);
  wk.expert = 0;
  wk.block = local / rows;
  wk.i0 = (first + local % rows) * BM;
  wk.i1 = min(wk.i0 + BM, a.places);
  return true;
}

// The row of x behind place i: its pair, as loaded, and the pair's token.  (The
// quotient of up to 2^22 by a float's reciprocal is off by one at most.)
__device__ __forceinline__ int mx4_pair(const Mx4Args& a, int i) { return a.order ? a.order[i] : i; }
__device__ __forceinline__ int mx4_row(const Mx4Args& a, int pair) {
  int row = pair;
  if (a.order) {
    row = (int)((float)pair * __builtin_amdgcn_rcpf((float)a.top_k));
    const int left = pair - row * a.top_k;
    row += (left >= a.top_k) - (left < 0);
  }
  return min(max(row, 0), a.x_rows - 1);
}

// Four columns c .. c + 3 of place p.
__device__ __forceinline__ void mx4_store(const Mx4Args& a, int p, int c, int cols_out, const mx4_f32x4& y) {
  const int64_t at = (int64_t)p * a.out_stride + c;
  if (c + 4 <= cols_out && a.out_vec) {
    if (a.out_dtype == HI_ROCM_DTYPE_BF16) {
      typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
      *reinterpret_cast<bf16x4*>((__bf16*)a.out + at) = __builtin_convertvector(y, bf16x4);
    } else {
      *reinterpret_cast<mx4_f32x4*>((float*)a.out + at) = y;
    }
    return;
  }
  #pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (c + q >= cols_out) break;
    if (a.out_dtype == HI_ROCM_DTYPE_BF16) ((__bf16*)a.out)[at + q] = (__bf16)y[q];
    else ((float*)a.out)[at + q] = y[q];
  }
}

// The scale of block b of place p; the last one's also sets those behind k.
__device__ __forceinline__ void mx4_store_scale(const Mx4Args& a, int p, int b, uint32_t s) {
  uint8_t* to = a.out_scales + (int64_t)p * a.out_scale_stride;
  to[mx4_scale_at(b)] = (uint8_t)s;
  if (b + 1 == a.cols / 2 / kMx4Block)
    for (int i = b + 1; i & 15; ++i) to[mx4_scale_at(i)] = 127;
}

// A block of 32 columns (from c, a multiple of 32) of place p as codes: lane 16
// g + r has columns 4 g .. + 3 of both halves.  All lanes of a place together.
__device__ __forceinline__ void mx4_store_codes(const Mx4Args& a, int p, bool in, int c, int g, const mx4_f32x4& lo,
                                                const mx4_f32x4& hi) {
  const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  uint32_t m = 0u;
  #pragma unroll
  for (int q = 0; q < 8; ++q) m = max(m, __float_as_uint(v[q]) & 0x7fffffffu);
  m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
  m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
  const uint32_t s = mx4_scale_of(m >> 23), codes = mx4_codes(v, s);
  if (!in) return;
  uint8_t* to = (uint8_t*)a.out + (int64_t)p * a.out_stride + c / 2 + 2 * g;
  *reinterpret_cast<uint16_t*>(to) = (uint16_t)codes;
  *reinterpret_cast<uint16_t*>(to + 8) = (uint16_t)(codes >> 16);
  if (g == 0) mx4_store_scale(a, p, c / kMx4Block, s);
}

// Few places (decode): the weights are what is read.  The workgroup's waves take
// the steps of k in turn; each streams 64 columns' blocks straight into registers,
// a step ahead, and multiplies them with up to 16 places.  Rounded rows of x come
// the same way; bf16 ones are rounded into LDS first, while the first weights are on
// their way (loads return in order: asked for in the loop, x would hold up every
// weight asked for before it).  The waves' sums are added in wave order.
// What hides the latency of a workgroup's beginning and end is the number of
// workgroups a CU holds: with two or four steps ahead (120 and 156 registers) a
// head of 151,936 x 4096 took 56 us, with one (six workgroups a CU) 55; 200 tokens'
// experts 44 and 47, with one 40; with eight (spilling) 66 and 42.
constexpr int kFewWaves = 4;
constexpr int kFewCols = 64;

// bytes from row to row of x in LDS: 16 rows' reads of a block meet all banks
__host__ __device__ __forceinline__ int few_code_stride(int steps) { return steps * 64 + 16; }
__host__ __device__ __forceinline__ int few_scale_stride(int quads) { return quads * 16 + 4; }

template <bool CODES>
__global__ void __launch_bounds__(64 * kFewWaves, 6) mx4_few_kernel(Mx4Args a) {
  extern __shared__ __align__(16) char few_smem[];
  constexpr int W = kFewWaves, COLS = kFewCols, NT = COLS / 16;
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols;
  const int per = a.swiglu ? COLS / 2 : COLS;
  MoeWork wk;
  if (!mx4_work<16>(a, (cols_out + per - 1) / per, wk)) return;
  // (all lanes' alike, which divisions in vector registers hide from the compiler)
  wk.expert = __builtin_amdgcn_readfirstlane(wk.expert);
  wk.block = __builtin_amdgcn_readfirstlane(wk.block);
  const int c0 = wk.block * per, n_places = wk.i1 - wk.i0;
  // bf16 rows: this thread's blocks of them, asked for before the weights
  const int blocks = a.k / kMx4Block, todo = CODES ? 0 : n_places * blocks;
  uint4 raw[4];
  auto raw_load = [&](int b) {
    const int j = b / blocks;
    const uint4* p = reinterpret_cast<const uint4*>(a.x + mx4_row(a, mx4_pair(a, wk.i0 + j)) * a.x_stride) + (b - j * blocks) * 4;
    #pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = p[i];
  };
  if (!CODES && tid < todo) raw_load(tid);
  // The weights by buffer loads, whose addresses are a lane's constant and scalars:
  // two halves of the tiles (with swiglu gate columns, then up columns), each tile
  // so many bytes behind its half's first.
  constexpr int HN = NT / 2;
  __amdgpu_buffer_rsrc_t wr[2], sr[2];
  int w_tile[NT], s_tile[NT];
  const int w_lane = lane * 16, s_lane = r * 16 + g * 4;
  #pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int tile = min(c0 / 16 + u * (a.swiglu ? cols_out / 16 : HN), a.tiles - 1);
    const int64_t at = (int64_t)wk.expert * a.tiles + tile;
    wr[u] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + at * a.steps * 1024), 0, -1, kBufferConfig);
    sr[u] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w_scales + at * a.quads * 256), 0, -1, kBufferConfig);
    #pragma unroll
    for (int i = 0; i < HN; ++i) {
      const int behind = min(i, a.tiles - 1 - tile);
      w_tile[u * HN + i] = behind * a.steps * 1024;
      s_tile[u * HN + i] = behind * a.quads * 256;
    }
  }
  mx4_f32x4 acc[NT];
  #pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = mx4_f32x4{0.f, 0.f, 0.f, 0.f};
  const uint8_t *xp = nullptr, *xs = nullptr;
  mx4_i32x4 wv[NT], xv;
  int ws[NT], xsc;
  auto load_w = [&](int step) {
    #pragma unroll
    for (int t = 0; t < NT; ++t) {
      wv[t] = __builtin_amdgcn_raw_buffer_load_b128(wr[t / HN], w_lane, w_tile[t] + step * 1024, 0);
      ws[t] = __builtin_amdgcn_raw_buffer_load_b32(sr[t / HN], s_lane, s_tile[t] + (step >> 2) * 256, 0);
    }
  };
  auto load_x = [&](int step) {
    if constexpr (CODES) {
      // (past k: the row's neighbours or scales, any code being finite, meet weights
      // of 0 and scales of 1)
      xv = *reinterpret_cast<const mx4_i32x4*>(xp + (int64_t)step * 64);
      xsc = *reinterpret_cast<const int*>(xs + (step >> 2) * 16);
    }
  };
  load_w(min(wid, a.steps - 1));
  if constexpr (CODES) {  // (behind the weights, which need no row's number)
    const int64_t row = mx4_row(a, mx4_pair(a, min(wk.i0 + r, wk.i1 - 1)));
    xp = a.x + row * a.x_stride + 16 * g;
    xs = a.x_scales + row * a.x_scale_stride + 4 * g;
    load_x(min(wid, a.steps - 1));
  }
  const int xc_stride = few_code_stride(a.steps), xs_stride = few_scale_stride(a.quads);
  char* const x_scales = few_smem + n_places * xc_stride;
  if constexpr (!CODES) {
    // (blocks behind k in its last step: zeros)
    const int tail = a.steps * 4 - blocks;
    for (int i = tid; i < n_places * tail; i += 64 * W) {
      const int j = i / tail, b = blocks + i - j * tail;
      *reinterpret_cast<uint4*>(few_smem + j * xc_stride + b * 16) = uint4{0u, 0u, 0u, 0u};
      x_scales[j * xs_stride + mx4_scale_at(b)] = 127;
    }
    for (int b = tid; b < todo; b += 64 * W) {
      const uint32_t s = mx4_scale_of(mx4_field(mx4_max_pair(mx4_max_pair(mx4_max_of(raw[0]), mx4_max_of(raw[1])),
                                                             mx4_max_pair(mx4_max_of(raw[2]), mx4_max_of(raw[3])))));
      const uint4 c = {mx4_codes(raw[0], s), mx4_codes(raw[1], s), mx4_codes(raw[2], s), mx4_codes(raw[3], s)};
      const int j = b / blocks, kb = b - j * blocks;
      if (b + 64 * W < todo) raw_load(b + 64 * W);
      *reinterpret_cast<uint4*>(few_smem + j * xc_stride + kb * 16) = c;
      x_scales[j * xs_stride + mx4_scale_at(kb)] = (char)s;
    }
    moe_wait_lds();  // (the weights stay on their way)
    moe_barrier();
  }
  const int rr = min(r, n_places - 1);
  const char* const xrow = few_smem + rr * xc_stride + g * 16;
  const char* const srow = x_scales + rr * xs_stride + g * 4;
  const int shift = (wid & 3) * 8;  // every step of this wave's is the same of its quad
  auto multiply = [&](int step) {
    mx4_i32x4 xc;
    int s;
    if constexpr (CODES) {
      xc = xv;
      s = xsc;
    } else {
      xc = *reinterpret_cast<const mx4_i32x4*>(xrow + step * 64);
      s = *reinterpret_cast<const int*>(srow + (step >> 2) * 16);
    }
    s = (int)((uint32_t)s >> shift);
    #pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] = mx4_mfma(wv[t], xc, acc[t], (int)((uint32_t)ws[t] >> shift), s);
  };
  int s = wid;
  for (; s + W < a.steps; s += W) {
    multiply(s);
    load_w(s + W);
    load_x(s + W);
  }
  if (s < a.steps) multiply(s);
  mx4_f32x4* const part = reinterpret_cast<mx4_f32x4*>(few_smem);
  if constexpr (!CODES) moe_barrier();  // (x's place; its reads are behind their products)
  #pragma unroll
  for (int t = 0; t < NT; ++t) part[(t * W + wid) * 64 + lane] = acc[t];
  __syncthreads();
  auto total = [&](int t) {
    mx4_f32x4 y = part[t * W * 64 + lane];
    #pragma unroll
    for (int w = 1; w < W; ++w) y += part[(t * W + w) * 64 + lane];
    return y;
  };
  const int p = wk.i0 + r;
  if (a.swiglu) {  // two tiles of gate and two of up: a block of codes
    if (wid > 0 || c0 >= cols_out) return;
    mx4_f32x4 y[2];
    #pragma unroll
    for (int t = 0; t < 2; ++t) {
      const mx4_f32x4 gate = total(t), up = total(NT / 2 + t);
      #pragma unroll
      for (int q = 0; q < 4; ++q) y[t][q] = moe_silu_mul(gate[q], up[q]);
    }
    if (a.out_dtype == HI_ROCM_DTYPE_MX4) {
      mx4_store_codes(a, p, p < wk.i1, c0, g, y[0], y[1]);
    } else if (p < wk.i1) {
      #pragma unroll
      for (int t = 0; t < 2; ++t) mx4_store(a, p, c0 + t * 16 + 4 * g, cols_out, y[t]);
    }
    return;
  }
  static_assert(NT == W, "a tile a wave");
  const int c = c0 + wid * 16 + 4 * g;
  if (p >= wk.i1 || c >= cols_out) return;
  mx4_f32x4 y = total(wid);
  if (a.bias != nullptr) {
    #pragma unroll
    for (int q = 0; q < 4; ++q) y[q] += c + q < cols_out ? a.bias[c + q] : 0.f;
  }
  mx4_store(a, p, c, cols_out, y);
}

// Many places (prompts, many requests): 32 MT places by 64 CW weight rows a workgroup
// of four waves, with MFMA 32x32x64 (lane 32 h + r: row r, block h of a half step; D
// rows 8 i + 4 h .. + 3 of column r in registers 4 i .. + 3).  CW waves have all of the
// places by 64 of the weight rows each, and 4 / CW such groups a stretch of k each, whose
// sums are added through LDS at the end.  Few columns a workgroup make more workgroups
// where there would be less than one a CU: what a CU fetches takes 0.8 us a quad of
// 256 rows (80 bytes a ns, however much is asked for ahead), with one of 64 rows 0.3.
//
// Weights go from memory straight to registers, where no other wave needs them,
// AHEAD steps ahead.  x goes through LDS a quad of steps at a time, filled by
// direct loads a quad ahead, with its scales; so there is a barrier a quad, and two
// workgroups a CU work through each other's beginnings, ends and waits.  Before the
// barrier each wave waits for its own loads of the quad that is read behind it:
// loads return in order, and at least 4 AHEAD of weights were started later.
// Behind it the other buffer is filled, whose reads all waves have waited for.
//
// A row of a quad is 256 bytes; its 16-byte chunk c lies at c ^ (row & 15), so that
// the reads of a chunk of 16 rows meet all banks.  A load writes 64 lanes x 16
// contiguous bytes; the lanes choose their global addresses so that the chunks land
// there.  Chunks of x past k hold what follows in memory (the next row, or the
// scales): any code is finite, and meets weights of 0 and scales of 1.
//
// 8,192 x 4,096 x 16,384: 264 to 299 us by the card, 3.7 to 4.2 PFLOP/s, the matrix cores
// busy half the time at some 1.65 GHz.  These instructions alone, on random data in
// registers, reach 6.1 (the card's power; 8.4 on zeros), 180 us, and the loop without them
// takes 207: the two overlap by about half.  With weights through LDS too 344 (eight waves in
// two phases) and 396 (256 x 256 a workgroup).
typedef float mx4_f32x16 __attribute__((ext_vector_type(16)));

template <int J>
__device__ __forceinline__ mx4_f32x16 mx4_mfma32(const mx4_i32x4& a, const mx4_i32x4& b, const mx4_f32x16& c, int sa,
                                                 int sb) {
  const mx4_i32x8 wa = __builtin_shufflevector(a, a, 0, 1, 2, 3, -1, -1, -1, -1);
  const mx4_i32x8 wb = __builtin_shufflevector(b, b, 0, 1, 2, 3, -1, -1, -1, -1);
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 4, 4, J, sa, J, sb);
}

constexpr int kMx4OutBytes = 8192;  // a wave's, for 32 places of 64 columns

template <int MT, int CW>
struct Mx4Tile {
  static constexpr int BM = 32 * MT, KG = 4 / CW;
  // Steps: more do not fit 256 registers where MT is 3 or 4, and with 4 fewer workgroups of
  // 32 places share a CU (128 experts, 2048 x 768, 12 and 32 places: 21.4 and 26.4 us, with
  // 2 20.6 and 24.8).
  static constexpr int AHEAD = 2;
  static constexpr int CODES = BM * 256, SCALES = CW * 1024;       // bytes of a quad's codes, of 64 CW rows' scales
  static constexpr int BUFFER = CODES + 2 * SCALES;
  static constexpr int ROWS = 4 * CW, L = BM / ROWS + 2;            // of a load, loads a thread and quad
  static constexpr int BYTES = std::max(std::max(KG * 2 * BUFFER, 4 * kMx4OutBytes), MT * (KG - 1) * CW * kMx4OutBytes);
  static_assert(64 * CW >= BM, "a row's scales a thread");
};

// 32 places of a wave's results at a time through its own LDS, so that 16 bytes a
// lane and a row's bytes next to each other are written: all of the 32 places' reads,
// then all of their stores (a read and its store after another: experts of 256 places,
// 2048 x 768, bf16 terms, 72 us where this takes 65).
// PAST: rows past the caches (mx4_past).
template <int MT, int KG, typename T, int COLS, bool PAST>
__device__ __forceinline__ void mx4_tile_store(const Mx4Args& a, mx4_f32x16 (&acc)[MT][2], char* mem, int p0, int i1,
                                               int c0, int cols_out, int lane, int group) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef T vec __attribute__((ext_vector_type(4)));
  constexpr int ES = sizeof(T), N = 16 / ES;              // values of a chunk
  constexpr int LANES = COLS / N, ROWS = 64 / LANES;      // lanes of a row, rows at a time
  const int r = lane & 31, h = lane >> 5, c = lane % LANES, j0 = lane / LANES, col = c0 + c * N;
  const bool whole = a.out_vec && c0 + COLS <= cols_out;  // (all lanes alike)
  #pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (m % KG != group) continue;
    const int first = p0 + m * 32;
    if (first >= i1) return;
    // row j of 64 values: the 16-byte chunk c at c ^ (j & 7)
    #pragma unroll
    for (int t = 0; t < COLS / 32; ++t)
      #pragma unroll
      for (int i = 0; i < 4; ++i) {
        const mx4_f32x4 y = {acc[m][t][4 * i], acc[m][t][4 * i + 1], acc[m][t][4 * i + 2], acc[m][t][4 * i + 3]};
        const int at = (t * 32 + i * 8 + h * 4) * ES;
        *reinterpret_cast<vec*>(mem + r * (64 * ES) + (((at >> 4) ^ (r & 7)) << 4 | (at & 15))) =
            __builtin_convertvector(y, vec);
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    u32x4 v[32 / ROWS];
    #pragma unroll
    for (int q = 0; q < 32 / ROWS; ++q) {
      const int j = q * ROWS + j0;
      v[q] = *reinterpret_cast<const u32x4*>(mem + j * (64 * ES) + (c ^ (j & 7)) * 16);
    }
    T* to = (T*)a.out + (int64_t)(first + j0) * a.out_stride + col;
    const int64_t step = ROWS * a.out_stride;
    if (whole) {
      #pragma unroll
      for (int q = 0; q < 32 / ROWS; ++q, to += step) {
        if (first + q * ROWS + j0 >= i1) break;
        if constexpr (PAST) __builtin_nontemporal_store(v[q], reinterpret_cast<u32x4*>(to));
        else *reinterpret_cast<u32x4*>(to) = v[q];
      }
    } else {
      #pragma unroll
      for (int q = 0; q < 32 / ROWS; ++q, to += step) {
        if (first + q * ROWS + j0 >= i1) break;
        #pragma unroll
        for (int e = 0; e < N; ++e) {
          if (col + e >= cols_out) break;
          if constexpr (ES == 2) reinterpret_cast<uint16_t*>(to)[e] = (uint16_t)(v[q][e >> 1] >> (e & 1) * 16);
          else reinterpret_cast<uint32_t*>(to)[e] = v[q][e];
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// A wave's results: with swiglu half 0 of acc is the gate and half 1 up.
template <int MT, int KG>
__device__ __forceinline__ void mx4_tile_out(const Mx4Args& a, mx4_f32x16 (&acc)[MT][2], char* mem, int p0, int i1,
                                             int c0, int cols_out, int lane, int group) {
  const int r = lane & 31, h = lane >> 5;
  if (a.swiglu) {
    #pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m % KG != group) continue;
      #pragma unroll
      for (int i = 0; i < 16; ++i) acc[m][0][i] = moe_silu_mul(acc[m][0][i], acc[m][1][i]);
    }
    if (a.out_dtype == HI_ROCM_DTYPE_MX4) {
      // the 32 columns are a block; a place's other half is lane ^ 32's
      #pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m % KG != group) continue;
        uint32_t most = 0u;
        #pragma unroll
        for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(acc[m][0][i]) & 0x7fffffffu);
        const auto both = __builtin_amdgcn_permlane32_swap(most, most, false, false);
        const uint32_t s = mx4_scale_of(max((uint32_t)both[0], (uint32_t)both[1]) >> 23);
        uint32_t mine[2];
        #pragma unroll
        for (int q = 0; q < 2; ++q) {
          float v[8];
          #pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = acc[m][0][q * 8 + i];
          mine[q] = mx4_codes(v, s);  // columns 16 q + 4 h .. + 3, then 8 on
        }
        // lane r gets columns 0 .. 15 of the place, lane 32 + r the others: the upper
        // lanes of the first change places with the lower ones of the second
        const auto all = __builtin_amdgcn_permlane32_swap(mine[0], mine[1], false, false);
        const int p = p0 + m * 32 + r;
        if (p < i1 && c0 < cols_out) {
          const uint32_t lo = all[0], hi = all[1];
          uint2 w;
          w.x = (lo & 0xffffu) | hi << 16;
          w.y = lo >> 16 | (hi & 0xffff0000u);
          *reinterpret_cast<uint2*>((uint8_t*)a.out + (int64_t)p * a.out_stride + c0 / 2 + 8 * h) = w;
          if (h == 0) mx4_store_scale(a, p, c0 / kMx4Block, s);
        }
      }
      return;
    }
  }
  auto store = [&](auto type) {
    using T = decltype(type);
    if (a.swiglu) mx4_tile_store<MT, KG, T, 32, false>(a, acc, mem, p0, i1, c0, cols_out, lane, group);
    else if (a.past) mx4_tile_store<MT, KG, T, 64, true>(a, acc, mem, p0, i1, c0, cols_out, lane, group);
    else mx4_tile_store<MT, KG, T, 64, false>(a, acc, mem, p0, i1, c0, cols_out, lane, group);
  };
  if (a.out_dtype == HI_ROCM_DTYPE_BF16) store(__bf16());
  else store(float());
}

template <int MT, int CW>
__device__ __forceinline__ void mx4_many_tile(const Mx4Args& a, const MoeWork& wk, char* smem0) {
  typedef Mx4Tile<MT, CW> Tile;
  constexpr int KG = Tile::KG, D = Tile::AHEAD, L = Tile::L, ROWS = Tile::ROWS, COLS = 64 * CW;
  const int tid = threadIdx.x & (COLS - 1), lane = tid & 63, r = lane & 31, h = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  // this group of waves: quads [quad0, quad1) of k, up to step `steps`
  const int group = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / COLS);
  const int per = (a.quads + KG - 1) / KG, quad0 = min(group * per, a.quads), quad1 = min(quad0 + per, a.quads);
  const int steps = min(quad1 * 4, a.steps);
  char* const smem = smem0 + group * 2 * Tile::BUFFER;
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols;
  const int expert = __builtin_amdgcn_readfirstlane(wk.expert), block = __builtin_amdgcn_readfirstlane(wk.block);
  // this wave's first column: with swiglu 32 of gate and the same of up
  const int c0 = block * (a.swiglu ? COLS / 2 : COLS) + wid * (a.swiglu ? 32 : 64);
  // Its weights: two halves of 32 rows (two tiles; past the last one, that again).
  __amdgpu_buffer_rsrc_t wr[2];
  int w_lane[2];
  #pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int tile = min(c0 / 16 + t * (a.swiglu ? cols_out / 16 : 2), a.tiles - 1);
    const int64_t at = (int64_t)expert * a.tiles + tile;
    wr[t] = __builtin_amdgcn_make_buffer_rsrc((void*)(a.w + at * a.steps * 1024), 0, -1, kBufferConfig);
    w_lane[t] = min(r >> 4, a.tiles - 1 - tile) * a.steps * 1024 + h * 256 + (r & 15) * 16;
  }
  // the scales of the weight row behind lane's place in the wave
  const int half = lane >> 5, tile_s = min(c0 / 16 + half * (a.swiglu ? cols_out / 16 : 2), a.tiles - 1);
  const uint8_t* const wsp =
      a.w_scales +
      ((int64_t)expert * a.tiles + min(tile_s + (lane >> 4 & 1), a.tiles - 1)) * a.quads * 256 + (lane & 15) * 16;
  // x: a round of loads takes 16 rows, this thread's chunk of one.  (The rows'
  // numbers are asked for before the first weights, and needed behind them.)
  const int jr = tid / 16;
  int pair[L - 2];
  #pragma unroll
  for (int i = 0; i < L - 2; ++i) pair[i] = mx4_pair(a, min(wk.i0 + i * ROWS + jr, wk.i1 - 1));
  const int pair_s = mx4_pair(a, min(wk.i0 + min(tid, Tile::BM - 1), wk.i1 - 1));
  __builtin_amdgcn_sched_barrier(0);
  mx4_i32x4 w[D][2][2];
  auto load_w = [&](int slot, int step) {
    const int at = min(step, steps - 1) * 1024;
    #pragma unroll
    for (int t = 0; t < 2; ++t)
      #pragma unroll
      for (int u = 0; u < 2; ++u) w[slot][t][u] = __builtin_amdgcn_raw_buffer_load_b128(wr[t], w_lane[t] + u * 512, at, 0);
  };
  #pragma unroll
  for (int d = 0; d < D; ++d) load_w(d, quad0 * 4 + d);
  __builtin_amdgcn_sched_barrier(0);
  const uint8_t* xp[L - 2];
  #pragma unroll
  for (int i = 0; i < L - 2; ++i) xp[i] = a.x + (int64_t)mx4_row(a, pair[i]) * a.x_stride + 16 * ((tid & 15) ^ ((i * ROWS + jr) & 15));
  const uint8_t* const sp = a.x_scales + (int64_t)mx4_row(a, pair_s) * a.x_scale_stride;
  auto fill = [&](int quad) {  // (past the last quad, that again, for a buffer that is not read)
    char* to = smem + (quad & 1) * Tile::BUFFER;
    const int at = min(quad, quad1 - 1);
    #pragma unroll
    for (int i = 0; i < L - 2; ++i)
      __builtin_amdgcn_global_load_lds((moe_global*)(xp[i] + (int64_t)at * 256), (moe_lds*)(to + i * CW * 1024 + wid * 1024), 16,
                                       0, 0);
    // (every thread one row's scales, past the tile's the last one's: no branch, behind
    // which the compiler would not know how many loads are on their way)
    __builtin_amdgcn_global_load_lds((moe_global*)(sp + (int64_t)at * 16), (moe_lds*)(to + Tile::CODES + wid * 1024), 16, 0,
                                     0);
    __builtin_amdgcn_global_load_lds((moe_global*)(wsp + (int64_t)at * 256),
                                     (moe_lds*)(to + Tile::CODES + Tile::SCALES + wid * 1024), 16, 0, 0);
  };
  mx4_f32x16 acc[MT][2];
  #pragma unroll
  for (int m = 0; m < MT; ++m)
    #pragma unroll
    for (int t = 0; t < 2; ++t)
      #pragma unroll
      for (int i = 0; i < 16; ++i) acc[m][t][i] = 0.f;
  fill(quad0);
  const char* const xrow = smem + r * 256;
  const char* const srow = smem + Tile::CODES + r * 16 + h * 4;
  int xs[MT][2], ws[2][2];
  mx4_i32x4 xf[2][MT];
  auto read_x = [&](const char* x, int half) {
    #pragma unroll
    for (int m = 0; m < MT; ++m)
      xf[half & 1][m] = *reinterpret_cast<const mx4_i32x4*>(x + m * 8192 + ((2 * half + h) ^ (r & 15)) * 16);
  };
  auto multiply = [&](auto j_, int u) {
    constexpr int J = decltype(j_)::value;
    #pragma unroll
    for (int m = 0; m < MT; ++m)
      #pragma unroll
      for (int t = 0; t < 2; ++t)
        acc[m][t] = mx4_mfma32<J>(w[J % D][t][u], xf[u][m], acc[m][t], ws[t][u], xs[m][u]);
  };
  auto step = [&](auto j_, int quad) {
    constexpr int J = decltype(j_)::value;
    const char* x = xrow + (quad & 1) * Tile::BUFFER;
    // this step's weights: all but the D - 1 newer steps', and what begin() started
    // since
    moe_wait_loads<4 * (D - 1) + (J < D ? L : 0)>();
    // a half's x is read while the half before it is multiplied (the first of a quad
    // by begin)
    read_x(x, 2 * J + 1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(j_, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (J < 3) read_x(x, 2 * J + 2);
    __builtin_amdgcn_sched_barrier(0);
    multiply(j_, 1);
    load_w(J % D, quad * 4 + J + D);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto begin = [&](int quad) {
    moe_wait<4 * D>();
    moe_barrier();
    fill(quad + 1);
    __builtin_amdgcn_sched_barrier(0);
    const char* sc = srow + (quad & 1) * Tile::BUFFER;
    #pragma unroll
    for (int u = 0; u < 2; ++u) {
      #pragma unroll
      for (int m = 0; m < MT; ++m) xs[m][u] = *reinterpret_cast<const int*>(sc + m * 512 + u * 8);
      #pragma unroll
      for (int t = 0; t < 2; ++t) ws[t][u] = *reinterpret_cast<const int*>(sc + Tile::SCALES + wid * 1024 + t * 512 + u * 8);
    }
    read_x(xrow + (quad & 1) * Tile::BUFFER, 0);
  };
  // Whole quads, without a condition that loads could be moved behind; the rest.
  // (begin() counts on the loads that a whole quad's steps started.  Those above may
  // be fewer: the compiler leaves out what a short k does not use.)
  moe_wait<0>();
  int quad = quad0;
  for (; quad < steps / 4; ++quad) {
    begin(quad);
    step(std::integral_constant<int, 0>(), quad);
    step(std::integral_constant<int, 1>(), quad);
    step(std::integral_constant<int, 2>(), quad);
    step(std::integral_constant<int, 3>(), quad);
  }
  if (quad < quad1) {
    begin(quad);
    step(std::integral_constant<int, 0>(), quad);
    if (quad * 4 + 1 < a.steps) step(std::integral_constant<int, 1>(), quad);
    if (quad * 4 + 2 < a.steps) step(std::integral_constant<int, 2>(), quad);
  }
  if constexpr (KG > 1)  // (as many barriers as the other groups)
    for (int i = quad1 - quad0; i < per; ++i) moe_barrier();
  moe_wait<0>();  // no load may still write LDS when it is used again, or the workgroup ends
  moe_barrier();
  if constexpr (KG > 1) {
    mx4_f32x4* const part = reinterpret_cast<mx4_f32x4*>(smem0);
    auto at = [&](int m, int g, int t, int i) { return (((m * (KG - 1) + g) * CW + wid) * 8 + t * 4 + i) * 64 + lane; };
    #pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m % KG == group) continue;
      #pragma unroll
      for (int t = 0; t < 2; ++t)
        #pragma unroll
        for (int i = 0; i < 4; ++i)
          part[at(m, group - (group > m % KG), t, i)] =
              mx4_f32x4{acc[m][t][4 * i], acc[m][t][4 * i + 1], acc[m][t][4 * i + 2], acc[m][t][4 * i + 3]};
    }
    __syncthreads();
    #pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (m % KG != group) continue;
      #pragma unroll
      for (int g = 0; g < KG - 1; ++g)
        #pragma unroll
        for (int t = 0; t < 2; ++t)
          #pragma unroll
          for (int i = 0; i < 4; ++i) {
            const mx4_f32x4 y = part[at(m, g, t, i)];
            #pragma unroll
            for (int q = 0; q < 4; ++q) acc[m][t][4 * i + q] += y[q];
          }
    }
    __syncthreads();
  }
  if (a.bias != nullptr) {
    #pragma unroll
    for (int t = 0; t < 2; ++t)
      #pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = c0 + t * 32 + i / 4 * 8 + h * 4 + i % 4;
        const float b = c < cols_out ? a.bias[c] : 0.f;
        #pragma unroll
        for (int m = 0; m < MT; ++m) acc[m][t][i] += b;
      }
  }
  mx4_tile_out<MT, KG>(a, acc, smem0 + (group * CW + wid) * kMx4OutBytes, wk.i0, wk.i1, c0, cols_out, lane, group);
}

// A tile of fewer places than its 32 MT is multiplied as one of fewer 32s.
template <int MT, int CW>
__global__ void __launch_bounds__(256, 2) mx4_many_kernel(Mx4Args a) {
  extern __shared__ __align__(16) char mx4_smem[];
  const int cols_out = a.swiglu ? a.cols / 2 : a.cols, per = a.swiglu ? 32 * CW : 64 * CW;
  MoeWork wk;
  if (!mx4_work<32 * MT>(a, (cols_out + per - 1) / per, wk)) return;
  const int need = (wk.i1 - wk.i0 + 31) / 32;
  if constexpr (MT > 1)
    if (need == 1) return mx4_many_tile<1, CW>(a, wk, mx4_smem);
  if constexpr (MT > 2)
    if (need == 2) return mx4_many_tile<2, CW>(a, wk, mx4_smem);
  if constexpr (MT > 3)
    if (need == 3) return mx4_many_tile<3, CW>(a, wk, mx4_smem);
  mx4_many_tile<MT, CW>(a, wk, mx4_smem);
}

int64_t mx4_grid(const Mx4Args& a, int bm, int bn) {
  if (a.offsets != nullptr) return moe_grid(a, bm, bn);
  const int64_t nt = ((int64_t)a.places + bm - 1) / bm;
  return (nt * (((int64_t)a.cols + bn - 1) / bn) + kXcds - 1) / kXcds * kXcds;
}

template <bool CODES>
hipError_t launch_few(const Mx4Args& a, hipStream_t st) {
  const int64_t grid = mx4_grid(a, 16, kFewCols);
  if (!moe_grid_fits(grid, 64 * kFewWaves)) return hipErrorInvalidConfiguration;
  int bytes = kFewCols / 16 * kFewWaves * 1024;  // the waves' sums, and before them x
  if (!CODES) bytes = std::max(bytes, std::min(a.places, 16) * (few_code_stride(a.steps) + few_scale_stride(a.quads)));
  auto* kernel = mx4_few_kernel<CODES>;
  const hipError_t e = ensure_lds((const void*)kernel, bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * kFewWaves), (unsigned)bytes, st, a);
  return hipGetLastError();
}

template <int MT, int CW>
hipError_t launch_many(const Mx4Args& a, hipStream_t st) {
  auto* kernel = mx4_many_kernel<MT, CW>;
  constexpr int bytes = Mx4Tile<MT, CW>::BYTES;
  const int64_t grid = mx4_grid(a, 32 * MT, 64 * CW);
  if (!moe_grid_fits(grid, 256)) return hipErrorInvalidConfiguration;
  const hipError_t e = ensure_lds((const void*)kernel, bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), (unsigned)bytes, st, a);
  return hipGetLastError();
}

// Which kernel, and its tile.  The time of a linear layer is taken as
//   max(fixed + rounds * quads * a quad's, weights at 5.8 TB/s + what is not hidden)
// us, a round being a workgroup on each CU (two of them on one take twice as long, and
// where there are many rounds, what counts is their average).  Measured, products
// alone, rows as given (f: the kernel for few; places x columns):
//   n 4,096, k 14,336   f 18.4 to 64; 32 x 256: 25, 32 x 128: 17, 32 x 64: 13 up to 128 rows;
//                       64 x 128: 23 at 512 rows, 64 x 256: 37 at 1,024, 128 x 256: 63 at 2,048
//   n 4,096, k 4,096    f 6.9, 8.7, 7.0, 6.4 at 32 rows; 256 rows 10.2, 9.0, 11.2 (32 x 256, 128, 64)
//   n 1,000, k 8,192    f 11, 15, 9.8, 8.2 at 32 rows; 512 rows 16.7, 11.8, 10.4
//   n 2,048, k 1,024    f 3.6, 4.8, 4.8, 5.2 at 32 rows
//   n 16,384, k 4,096   rows 128: 11, 13, 15, 19 (32, 64, 96, 128 places); 320: 27, 26, 17, 21; 512: 35, 25, 28, 23
//   n 16,384, k 8,192   f 13 to 16 rows, 20 above; 32 x 256, 128, 64: 17, 14, 15 at 16 rows
// Rows that come as bf16 only the first kernel takes (mx4_needs_rows, mx4_round_on_the_way).
//
// Experts with up to seven places each the first kernel always takes (128 experts, 1536 x
// 2048, 4, 8, 16 places: 31, 40, 52; 32 places a tile 34, 37, 42).  Of more the places are
// known on the device alone: experts are taken to fill three quarters of a tile more than
// their places, and rounds that are not whole to cost a half more.
//   128 experts, 1536 x 2048, 48 places each: 50, 45, 47, 49 (32 to 128 places x 256);
//     128: 85, 69, 61, 59; 256 (4,096 tokens x 8, with 2048 x 768, bf16 terms): 161 for both in
//     96 places, 150 in 128; 512: 242, 178, 160, 151
//   8 experts, 2048 x 4096, 24 places: 11.6, 10.2, 11.9 (32 x 256, 128, 64); f 12.7
//   60 experts, 1408 x 1440, 48 places: 15.9, 15.8, 18.4 (32, 64, 96 x 256); f 29
struct Mx4Shape {
  int mt, cw;
  float fixed, quad;  // us: of a launch, of a quad by a round of workgroups
};
constexpr Mx4Shape kMx4Shapes[] = {{4, 4, 2.5f, 2.25f}, {3, 4, 2.5f, 1.9f}, {2, 4, 2.5f, 1.5f}, {1, 4, 2.5f, 1.05f},
                                   {2, 2, 3.5f, 0.85f}, {1, 2, 3.5f, 0.6f}, {1, 1, 3.9f, 0.4f}};
constexpr float kFewFixed = 2.6f, kFewQuad = 0.56f, kManyHidden = 2.5f, kMx4Rate = 5.8e6f;  // bytes a us

// Quads of k by rounds of workgroups of bm places by bn columns.
float mx4_rounds(const Mx4Args& a, int bm, int bn) {
  const bool grouped = a.offsets != nullptr;
  const int64_t met = std::min(a.experts, a.places);
  const int64_t tiles = grouped ? std::max(met, a.places / bm + met * 3 / 4) : ((int64_t)a.places + bm - 1) / bm;
  const int64_t wgs = tiles * (((int64_t)a.cols + bn - 1) / bn);
  if (wgs <= 256) return (float)a.quads;
  const float r = (float)wgs / 256.f;
  return (float)a.quads * (grouped ? r + 0.5f : wgs <= 1024 ? std::ceil(r) : r);
}

struct Mx4Choice {
  Mx4Shape shape;  // mt 0: the kernel for few
  float us;
};
Mx4Choice mx4_choose(const Mx4Args& a) {
  const Mx4Shape few = {0, 1, kFewFixed, kFewQuad};
  const bool grouped = a.offsets != nullptr;
  if (grouped && a.places / a.experts < 8) return {few, 0.f};
  const float read = grouped ? 0.f : (float)a.tiles * 16.f * (float)a.k * (17.f / 32.f) / kMx4Rate;
  Mx4Choice best = {kMx4Shapes[0], INFINITY};
  for (const Mx4Shape& s : kMx4Shapes) {
    const float t = std::max(s.fixed + mx4_rounds(a, 32 * s.mt, 64 * s.cw) * s.quad, read + kManyHidden);
    if (t < best.us) best = {s, t};
  }
  const float t = std::max(few.fixed + mx4_rounds(a, 16, kFewCols) * few.quad, read);
  if (t < best.us) best = {few, t};
  return best;
}

// Whether more bf16 rows than 16 (up to 4,096 inputs: mx4_few_kernel's LDS) are rounded by
// the workgroups that multiply them rather than beforehand, which is another launch of
// 2.5 us: theirs take 2.8 + 0.7 a quad and round, and x from the L2s at 20 TB/s.  17 to 64
// rows, us in a graph (eagerly another 4 for the second launch): 512 x 512 3.3 against 5.5, 2,048
// x 1,024 4.2 and 6.3, 8,192 x 1,024 4.2 to 5.6 and 6.4 to 7.2, 4,096 x 2,048 5.7 and 7.5;
// 4,096 x 4,096 17 rows 8.9 and 9.8, 64 rows 10.8 and 9.9; 32,000 x 1,024 64 rows 13.5 and 9.8.
bool mx4_round_on_the_way(const Mx4Args& a) {
  if (a.offsets != nullptr || a.k > 4096) return false;
  const float wgs = (float)(((int64_t)a.places + 15) / 16 * (((int64_t)a.cols + kFewCols - 1) / kFewCols));
  return 2.8f + mx4_rounds(a, 16, kFewCols) * 0.7f + wgs * 32.f * (float)a.k / 20e6f < mx4_choose(a).us + 2.5f;
}

hipError_t launch_product(const Mx4Args& a, bool codes, hipStream_t st) {
  if (!codes) return launch_few<false>(a, st);
  const Mx4Shape s = mx4_choose(a).shape;
  switch (s.mt * 8 + s.cw) {
    case 1: return launch_few<true>(a, st);
    case 12: return launch_many<1, 4>(a, st);
    case 20: return launch_many<2, 4>(a, st);
    case 28: return launch_many<3, 4>(a, st);
    case 18: return launch_many<2, 2>(a, st);
    case 10: return launch_many<1, 2>(a, st);
    case 9: return launch_many<1, 1>(a, st);
    default: return launch_many<4, 4>(a, st);
  }
}

// Whether a linear layer's tiles store their results past the caches: where the last-level
// cache does not hold them (256 MB), so that x and the weights stay there, and between one
// L2 and all eight, whose dirty lines a launch's end writes back.  Elsewhere what reads the
// result next loses more than the product gains.  us with and without, layers of k 4,096 on
// end, alone and each with the rounding of its result:
//   1.0 MB (128 x 4,096 bf16)      7.3 and 7.2, 10.5 and 10.1
//   2.6 MB (320 x 4,096 bf16)      10.1 and 10.2, 13.4 and 13.2
//   5.2 MB (320 x 4,096 f32)       10.5 and 10.5, 14.3 and 14.4
//   10.5 MB (320 x 16,384 bf16)    16.9 and 17.9, 21.8 and 22.0
//   16.8 MB (2,048 x 4,096 bf16)   19.8 and 21.1, 25.5 and 26.2
//   33.6 MB (2,048 x 4,096 f32)    22.6 and 23.4, 30.8 and 30.7
//   67 MB (1,024 x 16,384 f32)     45.8 and 44.8, 60.4 and 57.1
//   134 MB (8,192 x 4,096 f32)     72.8 and 76.8, 104 and 99.6
//   197 MB (6,000 x 16,384 bf16)   206 and 207, 245 and 240
//   249 MB (7,600 x 16,384 bf16)   260 and 261, 307 and 309
//   268 MB (8,192 x 16,384 bf16)   283 and 290, 337 and 343
//   537 MB (8,192 x 16,384 f32)    321 and 342, 425 and 460
// (The experts' terms, 67 and 134 MB at 4,096 tokens, are read next.)
constexpr double kMx4PastOne = 4e6, kMx4PastAll = 32e6, kMx4PastLast = 240e6;
bool mx4_past(int64_t rows, int n, int size) {
  const double bytes = (double)rows * n * size;
  return (bytes > kMx4PastOne && bytes <= kMx4PastAll) || bytes > kMx4PastLast;
}

bool mx4_float(int d) { return d == HI_ROCM_DTYPE_F32 || d == HI_ROCM_DTYPE_BF16; }
int mx4_size(int d) { return d == HI_ROCM_DTYPE_F32 ? 4 : 2; }

// Few bf16 rows are rounded by each workgroup in LDS, at most 16 of them and 65,536
// values (36 KB); more, beforehand in a workspace, but for mx4_round_on_the_way.
bool mx4_needs_rows(int64_t x_rows, int64_t places, int k) {
  return x_rows > 16 || std::min<int64_t>(places, 16) * k > 65536;
}

// A linear layer's rows: the weight and the number of rows are in `a`.
bool mx4_linear_needs_rows(const Mx4Args& a) {
  return mx4_needs_rows(a.places, a.places, a.k) && !mx4_round_on_the_way(a);
}

// x as a product reads it: "rows" given, bf16 rows as they are when they are
// few, or "rows" made of them in the workspace.
int mx4_take_x(const char* name, Mx4Args& a, const void* x, int x_dtype, int64_t x_rows, int64_t x_stride, bool needs,
               void* ws, hipStream_t st, bool& codes) {
  const Mx4Rows L = mx4_rows_layout(x_rows, a.k);
  a.x_rows = (int)x_rows;
  codes = x_dtype == HI_ROCM_DTYPE_MX4 || needs;
  if (!codes) {
    a.x = (const uint8_t*)x;
    a.x_stride = x_stride * 2;
    return HI_ROCM_OK;
  }
  if (x_dtype != HI_ROCM_DTYPE_MX4) {
    const hipError_t e = mx4_make_rows(x, x_dtype, x_rows, a.k, x_stride, ws, st);
    if (e != hipSuccess) return api_hip_fail(e, name);
    x = ws;
  }
  a.x = (const uint8_t*)x;
  a.x_stride = L.code_stride;
  a.x_scales = (const uint8_t*)x + L.scales;
  a.x_scale_stride = L.scale_stride;
  return HI_ROCM_OK;
}

int mx4_fail(int status, const char* name, const char* what) {
  char text[256];
  snprintf(text, sizeof(text), "%s: %s", name, what);
  return api_fail(status, text);
}

// What both products check of x, the weight and the workspace.
int mx4_check(const char* name, const void* x, int x_dtype, int64_t x_rows, int64_t x_stride, const void* packed,
              size_t packed_bytes, int experts, int n, int k) {
  if (x == nullptr || packed == nullptr || x_rows <= 0 || n <= 0 || k <= 0 || experts <= 0 ||
      (x_dtype != HI_ROCM_DTYPE_BF16 && x_dtype != HI_ROCM_DTYPE_MX4) || (x_dtype == HI_ROCM_DTYPE_BF16 && x_stride < k))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "invalid arguments");
  if (!mx4_weight_fits(experts, n, k) || x_rows > HI_ROCM_MX4_MAX_ROWS)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name,
                    "needs k a multiple of 32 up to 2^24, at most 2048 experts, 2^24 outputs, 2^35 weights, 2^22 rows");
  if ((uintptr_t)packed % 16 != 0 || packed_bytes < mx4_packed_layout(experts, n, k).total)
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "packed not on 16 bytes, or too small (hi_rocm_mx4_packed_bytes)");
  if ((uintptr_t)x % 16 != 0 || (x_dtype == HI_ROCM_DTYPE_BF16 && x_stride % 8 != 0))
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "needs rows that start on 16 bytes");
  return HI_ROCM_OK;
}
int mx4_check_workspace(const char* name, int x_dtype, bool needs, int64_t x_rows, int k, const void* ws, size_t ws_bytes) {
  if (x_dtype == HI_ROCM_DTYPE_BF16 && needs &&
      (ws == nullptr || (uintptr_t)ws % 16 != 0 || ws_bytes < mx4_rows_layout(x_rows, k).total))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "workspace not on 16 bytes, or too small (hi_rocm_mx4_workspace_bytes)");
  return HI_ROCM_OK;
}

void mx4_take_weight(Mx4Args& a, const void* packed, int experts, int n, int k) {
  const Mx4Packed L = mx4_packed_layout(experts, n, k);
  a.w = (const uint8_t*)packed;
  a.w_scales = (const uint8_t*)packed + L.scales;
  a.experts = experts;
  a.cols = n;
  a.k = k;
  a.tiles = (int)L.tiles;
  a.steps = (int)L.steps;
  a.quads = (int)L.quads;
}

}  // namespace
}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_mx4_workspace_bytes(int x_rows, int places, int k, size_t* out_bytes) {
  if (x_rows <= 0 || places <= 0 || k <= 0 || out_bytes == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_workspace_bytes: invalid arguments");
  if (k % kMx4Block != 0 || k > HI_ROCM_MX4_MAX_K || x_rows > HI_ROCM_MX4_MAX_ROWS || places > HI_ROCM_MX4_MAX_ROWS)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_mx4_workspace_bytes: needs k a multiple of 32 up to 2^24, at most 2^22 rows and places");
  *out_bytes = mx4_needs_rows(x_rows, places, k) ? mx4_rows_layout(x_rows, k).total : 0;
  return HI_ROCM_OK;
}

int hi_rocm_mx4_linear_workspace_bytes(int rows, int n, int k, size_t* out_bytes) {
  if (rows <= 0 || n <= 0 || k <= 0 || out_bytes == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_mx4_linear_workspace_bytes: invalid arguments");
  if (!mx4_weight_fits(1, n, k) || rows > HI_ROCM_MX4_MAX_ROWS)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_mx4_linear_workspace_bytes: needs k a multiple of 32 up to 2^24, at most 2^24 outputs, 2^35 "
                    "weights, 2^22 rows");
  Mx4Args a;
  memset(&a, 0, sizeof(a));
  mx4_take_weight(a, nullptr, 1, n, k);
  a.places = rows;
  *out_bytes = mx4_linear_needs_rows(a) ? mx4_rows_layout(rows, k).total : 0;
  return HI_ROCM_OK;
}

int hi_rocm_debug_mx4_linear(int rows, int n, int k, int x_dtype, int out_dtype, int* out_places, int* out_cols,
                             int* out_past) {
  if (rows <= 0 || n <= 0 || k <= 0 || (x_dtype != HI_ROCM_DTYPE_BF16 && x_dtype != HI_ROCM_DTYPE_MX4) ||
      !mx4_float(out_dtype) || out_places == nullptr || out_cols == nullptr || out_past == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_debug_mx4_linear: invalid arguments");
  if (!mx4_weight_fits(1, n, k) || rows > HI_ROCM_MX4_MAX_ROWS)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_debug_mx4_linear: needs k a multiple of 32 up to 2^24, at most 2^24 outputs, 2^35 weights, "
                    "2^22 rows");
  Mx4Args a;
  memset(&a, 0, sizeof(a));
  mx4_take_weight(a, nullptr, 1, n, k);
  a.places = rows;
  const bool codes = x_dtype == HI_ROCM_DTYPE_MX4 || mx4_linear_needs_rows(a);
  const Mx4Shape s = mx4_choose(a).shape;
  const bool many = codes && s.mt > 0;
  *out_places = many ? 32 * s.mt : 16;
  *out_cols = many ? 64 * s.cw : kFewCols;
  *out_past = many && mx4_past(rows, n, mx4_size(out_dtype));
  return HI_ROCM_OK;
}

int hi_rocm_mx4_linear(const void* x, int x_dtype, int rows, int64_t x_stride, const void* packed, size_t packed_bytes,
                       int n, int k, const float* bias, void* out, int out_dtype, int64_t out_stride, void* workspace,
                       size_t workspace_bytes, void* stream) {
  const char* name = "hi_rocm_mx4_linear";
  int bad = mx4_check(name, x, x_dtype, rows, x_stride, packed, packed_bytes, 1, n, k);
  if (bad != HI_ROCM_OK) return bad;
  if (out == nullptr || !mx4_float(out_dtype) || out_stride < n || (uintptr_t)out % mx4_size(out_dtype) != 0 ||
      (uintptr_t)bias % 4 != 0)
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "invalid arguments");
  Mx4Args a;
  memset(&a, 0, sizeof(a));
  mx4_take_weight(a, packed, 1, n, k);
  a.places = rows;
  const bool needs = mx4_linear_needs_rows(a);
  bad = mx4_check_workspace(name, x_dtype, needs, rows, k, workspace, workspace_bytes);
  if (bad != HI_ROCM_OK) return bad;
  a.bias = bias;
  a.out = out;
  a.out_stride = out_stride;
  a.out_dtype = out_dtype;
  a.out_vec = (uintptr_t)out % 16 == 0 && out_stride * mx4_size(out_dtype) % 16 == 0;
  a.past = mx4_past(rows, n, mx4_size(out_dtype));
  a.top_k = 1;
  bool codes;
  const int rc = mx4_take_x(name, a, x, x_dtype, rows, x_stride, needs, workspace, (hipStream_t)stream, codes);
  if (rc != HI_ROCM_OK) return rc;
  const hipError_t e = launch_product(a, codes, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "too many rows and outputs for one launch");
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 linear launch");
}

int hi_rocm_mx4_grouped_product(const void* x, int x_dtype, int x_rows, int64_t x_stride, const int32_t* order,
                                int top_k, const int32_t* offsets, int places, int experts, const void* packed,
                                size_t packed_bytes, int cols, int k, int swiglu, void* out, int out_dtype,
                                int64_t out_stride, size_t out_bytes, void* workspace, size_t workspace_bytes,
                                void* stream) {
  const char* name = "hi_rocm_mx4_grouped_product";
  int bad = mx4_check(name, x, x_dtype, x_rows, x_stride, packed, packed_bytes, experts, cols, k);
  if (bad != HI_ROCM_OK) return bad;
  const bool needs = mx4_needs_rows(x_rows, places, k);
  bad = mx4_check_workspace(name, x_dtype, needs, x_rows, k, workspace, workspace_bytes);
  if (bad != HI_ROCM_OK) return bad;
  const int wide = swiglu ? cols / 2 : cols;
  const bool to_rows = out_dtype == HI_ROCM_DTYPE_MX4;
  if (offsets == nullptr || out == nullptr || places <= 0 || (order && top_k <= 0) || (!order && x_rows < places) ||
      (!to_rows && (!mx4_float(out_dtype) || out_stride < wide || (uintptr_t)out % mx4_size(out_dtype) != 0)) ||
      (to_rows && !swiglu))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "invalid arguments");
  if (swiglu && cols % 64 != 0)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "needs gate and up halves of a multiple of 32 columns");
  if (places > HI_ROCM_MX4_MAX_ROWS)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "more than 2^22 places");
  if (to_rows && ((uintptr_t)out % 16 != 0 || out_bytes < mx4_rows_layout(places, wide).total))
    return mx4_fail(HI_ROCM_ERR_ARGS, name, "out not on 16 bytes, or too small (hi_rocm_mx4_rows_bytes)");
  Mx4Args a;
  memset(&a, 0, sizeof(a));
  mx4_take_weight(a, packed, experts, cols, k);
  a.order = order;
  a.offsets = offsets;
  a.out = out;
  a.out_stride = out_stride;
  a.out_dtype = out_dtype;
  if (to_rows) {
    const Mx4Rows L = mx4_rows_layout(places, wide);
    a.out_stride = L.code_stride;
    a.out_scales = (uint8_t*)out + L.scales;
    a.out_scale_stride = L.scale_stride;
  } else {
    a.out_vec = (uintptr_t)out % 16 == 0 && out_stride * mx4_size(out_dtype) % 16 == 0;
  }
  a.places = places;
  a.top_k = order ? top_k : 1;
  a.swiglu = swiglu != 0;
  bool codes;
  const int rc = mx4_take_x(name, a, x, x_dtype, x_rows, x_stride, needs, workspace, (hipStream_t)stream, codes);
  if (rc != HI_ROCM_OK) return rc;
  const hipError_t e = launch_product(a, codes, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return mx4_fail(HI_ROCM_ERR_UNSUPPORTED, name, "too many places and columns for one launch");
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "mx4 grouped product launch");
}

}  // extern "C"
