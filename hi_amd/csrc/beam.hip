// Beam search: the selection over a request's beams and the vocabulary, and
// the reordering of the beams' states.  (The reference decodes without beams;
// no counterpart there.)
//
// Selection.  For a beam with cumulative log-probability c and logits l over
// its allowed tokens (NaN logits count as masked):
//     lse = m + log sum_v exp(l_v - m),  m = max_v l_v
//     score(v) = c + (l_v - lse)
// each a single f32 rounding but the sum, and a request keeps the first n_out
// candidates of all its beams in the order (score descending, beam ascending,
// logit descending, token ascending).  Within a beam that is the order of the
// logits, so a part of a row can keep its n_out first candidates without
// knowing lse, and no rounding of a score decides between two tokens of a
// beam.
//
// Two kernels read each logit once:
//  * beam_part_kernel: a part of a row in registers: its maximum, its sum of
//    exponentials, and its first n_out candidates by (logit, token);
//  * beam_finish_kernel: a request: its beams' lse from the parts, and the
//    first n_out of the parts' candidates.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "hi_rocm.h"
#include "sampler_internal.h"
#include "wave_ops.h"

namespace hi_rocm {
namespace {

constexpr int kBeamMax = HI_ROCM_BEAM_MAX;
constexpr int kBeamMaxOut = HI_ROCM_BEAM_MAX_OUT;
constexpr int kPartThreads = 256;
constexpr int kPartSlots = 256;      // candidates a part can hold before it ranks them
constexpr int kFinishThreads = 1024;
constexpr int kFinishSlots = 512;
constexpr int kBeamMaxRows = 65536;

struct BeamPart {
  float m;       // largest logit of the part (-inf: no candidate)
  float sum;     // sum of exp(l - m)
  uint32_t n;    // candidates kept
  uint32_t pad;
};

struct BeamArgs {
  const void* logits;
  int64_t row_stride;         // elements
  const float* scores;        // [rows]
  const uint8_t* finished;    // [rows] or null
  const uint32_t* mask;       // [rows][mask_words] or null
  int V, K, n_out, n_parts, mask_words;
  uint32_t eos;
  BeamPart* parts;            // [rows][n_parts]
  uint64_t* cand;             // [rows][n_parts][n_out], descending
  float* out_scores;          // [batch][n_out]
  uint32_t* out_tokens;
  int32_t* out_parents;
  uint8_t* out_finished;
};

__device__ __forceinline__ bool beam_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Order-preserving u32 of a non-NaN float, -0 as +0.
__device__ __forceinline__ uint32_t beam_okey(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float beam_okey_inv(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
constexpr uint32_t kBeamNegInf = 0x007fffffu;  // beam_okey(-inf): keys above it are candidates

__device__ __forceinline__ float beam_wave_max(float v) {
  #pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float beam_wave_sum(float v) {
  #pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// Whether a row takes part: a beam whose score is not finite has no
// candidates, a finished one has a single candidate that needs no logits.
__device__ __forceinline__ bool beam_reads(const BeamArgs& a, int row) {
  return beam_finite(a.scores[row]) && !(a.finished && a.finished[row]);
}

// The n-th largest key of G a lane over the wave (0 when fewer are above 0),
// bit by bit.
template <int G>
__device__ __forceinline__ uint32_t beam_wave_nth(const uint32_t (&key)[G], int n) {
  uint32_t t = 0u;
  #pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit != 0u; bit >>= 1) {
    const uint32_t c = t | bit;
    int cnt = 0;
    #pragma unroll
    for (int g = 0; g < G; ++g) cnt += __popcll(__ballot(key[g] >= c));
    if (cnt >= n) t = c;
  }
  return t;
}

// A bound with at least n keys of the workgroup (W waves, G keys a lane) at
// or above it: the smallest of the waves' ceil(n / W)-th keys, or the largest
// of their n-th.
template <int G, int W>
__device__ __forceinline__ uint32_t beam_bound(const uint32_t (&key)[G], int n, uint32_t* red) {
  const uint32_t share = beam_wave_nth<G>(key, (n + W - 1) / W);
  const uint32_t full = beam_wave_nth<G>(key, n);
  const int wid = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) { red[wid] = share; red[W + wid] = full; }
  __syncthreads();
  uint32_t lo = red[0], hi = red[W];
  #pragma unroll
  for (int w = 1; w < W; ++w) { lo = min(lo, red[w]); hi = max(hi, red[W + w]); }
  return max(lo, hi);
}

// 16 bytes of a row as floats.
template <int DT>
struct BeamLoad;
template <>
struct BeamLoad<HI_ROCM_DTYPE_F32> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float get(const i32x4_t& v, int q) { return __int_as_float(v[q]); }
};
template <>
struct BeamLoad<HI_ROCM_DTYPE_BF16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float get(const i32x4_t& v, int q) {
    const uint32_t w = (uint32_t)v[q >> 1];
    return __uint_as_float((q & 1) ? (w & 0xffff0000u) : (w << 16));
  }
};

// One part: kPartThreads * PER elements of a row, counted from the 16-byte
// boundary at or before the row's start (rows start anywhere; the elements
// before the start and after the end are no candidates).
template <int DT, int PER>
__global__ void __launch_bounds__(kPartThreads) beam_part_kernel(BeamArgs a) {
  constexpr int N = BeamLoad<DT>::N, L = PER / N, W = kPartThreads / 64, ES = 16 / N;
  constexpr int G = 4;  // groups a thread for the bound
  static_assert(PER % G == 0, "groups");
  __shared__ uint64_t slots[kPartSlots];
  __shared__ uint64_t red64[W];
  __shared__ uint32_t red[2 * W];
  __shared__ float redf[W];
  __shared__ uint32_t counter;
  const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  if (!beam_reads(a, row)) return;
  const char* p0 = (const char*)a.logits + (int64_t)row * a.row_stride * ES;
  const int head = (int)((uintptr_t)p0 & 15) / ES;
  const int64_t base = (int64_t)part * (kPartThreads * PER);  // elements from the aligned start
  // range-checked loads: bytes from this part's start to the row's end
  const int64_t left = ((int64_t)a.V + head - base) * ES;  // (the last part may lie after the row: nothing)
  constexpr int64_t kSpan = (int64_t)kPartThreads * PER * ES;
  const int bytes = left < 0 ? 0 : (int)(left < kSpan ? left : kSpan);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p0 - head * ES + base * ES), 0, (bytes + 3) & ~3, kBufferConfig);
  float x[PER];
  {
    i32x4_t v[L];
    #pragma unroll
    for (int j = 0; j < L; ++j) v[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, (j * kPartThreads + tid) * 16, 0, 0);
    #pragma unroll
    for (int j = 0; j < L; ++j) {
      #pragma unroll
      for (int q = 0; q < N; ++q) x[j * N + q] = BeamLoad<DT>::get(v[j], q);
    }
  }
  const float ninf = -__builtin_inff();
  // token of x[j * N + q]: t0 + j * kPartThreads * N + q
  const int t0 = (int)base + tid * N - head;
  const uint32_t* mrow = a.mask ? a.mask + (int64_t)row * a.mask_words : nullptr;
  #pragma unroll
  for (int j = 0; j < L; ++j) {
    const int t = t0 + j * (kPartThreads * N);
    uint64_t bits = ~0ull;
    if (mrow) {
      const int tc = t < 0 ? 0 : t, w = tc >> 5;
      const uint64_t lo = w < a.mask_words ? mrow[w] : 0u, hi = w + 1 < a.mask_words ? mrow[w + 1] : 0u;
      bits = ((hi << 32) | lo) >> (tc & 31);
      if (t < 0) bits <<= -t;
    }
    #pragma unroll
    for (int q = 0; q < N; ++q) {
      const float f = x[j * N + q];
      const bool ok = t + q >= 0 && t + q < a.V && f == f && ((bits >> q) & 1ull);
      x[j * N + q] = ok ? f : ninf;
    }
  }
  float gm[G];
  #pragma unroll
  for (int g = 0; g < G; ++g) {
    gm[g] = x[g * (PER / G)];
    #pragma unroll
    for (int i = 1; i < PER / G; ++i) gm[g] = fmaxf(gm[g], x[g * (PER / G) + i]);
  }
  float m = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
  m = beam_wave_max(m);
  if (lane == 0) redf[wid] = m;
  if (tid == 0) counter = 0u;
  __syncthreads();
  #pragma unroll
  for (int w = 0; w < W; ++w) m = fmaxf(m, redf[w]);
  const int64_t slot = (int64_t)row * a.n_parts + part;
  if (!beam_finite(m)) {  // nothing allowed, or a +inf logit: the finish sees which
    if (tid == 0) a.parts[slot] = BeamPart{m, 0.f, 0u, 0u};
    return;
  }
  float s = 0.f;
  #pragma unroll
  for (int i = 0; i < PER; ++i) s += __expf(x[i] - m);
  s = beam_wave_sum(s);
  // the part's candidates: all logits at or above a bound that n_out of them reach
  uint32_t key[G];
  #pragma unroll
  for (int g = 0; g < G; ++g) key[g] = beam_okey(gm[g]);
  const uint32_t bound = max(beam_bound<G, W>(key, a.n_out, red), kBeamNegInf + 1u);
  __syncthreads();
  if (lane == 0) redf[wid] = s;
  #pragma unroll
  for (int j = 0; j < L; ++j) {
    #pragma unroll
    for (int q = 0; q < N; ++q) {
      const uint32_t k = beam_okey(x[j * N + q]);
      if (k >= bound) {
        const uint32_t o = atomicAdd(&counter, 1u);
        if (o < (uint32_t)kPartSlots)
          slots[o] = ((uint64_t)k << 32) | (0xffffffffu - (uint32_t)(t0 + j * (kPartThreads * N) + q));
      }
    }
  }
  __syncthreads();
  const int n = (int)counter;
  uint64_t* out = a.cand + slot * a.n_out;
  const int keep = min(n, a.n_out);
  if (tid == 0) {
    s = redf[0];
    #pragma unroll
    for (int w = 1; w < W; ++w) s += redf[w];
    a.parts[slot] = BeamPart{m, s, (uint32_t)keep, 0u};
  }
  if (n <= kPartSlots) {
    // rank by counting
    if (tid < n) {
      const uint64_t mine = slots[tid];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += slots[i] > mine;
      if (rank < a.n_out) out[rank] = mine;
    }
    return;
  }
  // many equal logits: one candidate after another
  uint64_t prev = ~0ull;
  for (int r = 0; r < keep; ++r) {
    uint64_t best = 0ull;
    #pragma unroll
    for (int j = 0; j < L; ++j) {
      #pragma unroll
      for (int q = 0; q < N; ++q) {
        const uint64_t k = ((uint64_t)beam_okey(x[j * N + q]) << 32) |
                           (0xffffffffu - (uint32_t)(t0 + j * (kPartThreads * N) + q));
        if (k < prev && k > best) best = k;
      }
    }
    #pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t w = ((uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(best >> 32), o, 64) << 32) |
                         (uint32_t)__shfl_xor((int)(uint32_t)best, o, 64);
      best = w > best ? w : best;
    }
    if (lane == 0) red64[wid] = best;
    __syncthreads();
    best = red64[0];
    #pragma unroll
    for (int w = 1; w < W; ++w) best = red64[w] > best ? red64[w] : best;
    __syncthreads();
    prev = best;
    if (tid == 0) out[r] = best;
  }
}

// A candidate of a request: (score, beam) and (logit, token), both descending
// keys with the lower beam and token first.
struct BeamCand {
  uint64_t hi, lo;
};
__device__ __forceinline__ bool beam_before(const BeamCand& x, const BeamCand& y) {
  return x.hi > y.hi || (x.hi == y.hi && x.lo > y.lo);
}

__global__ void __launch_bounds__(kFinishThreads) beam_finish_kernel(BeamArgs a) {
  constexpr int W = kFinishThreads / 64;
  __shared__ BeamCand slots[kFinishSlots];
  __shared__ BeamCand redc[W];
  __shared__ float lse[kBeamMax];
  __shared__ uint32_t state[kBeamMax];  // 0: no candidates, 1: its parts' candidates, 2: finished
  __shared__ uint32_t red[2 * W];
  __shared__ uint32_t counter;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int row0 = b * a.K;
  const float ninf = -__builtin_inff();
  if (tid == 0) counter = 0u;
  for (int k = wid; k < a.K; k += W) {
    const int row = row0 + k;
    const float c = a.scores[row];
    uint32_t st = 0u;
    float l = 0.f;
    if (beam_finite(c)) {
      if (a.finished && a.finished[row]) {
        st = 2u;
      } else {
        const BeamPart* pp = a.parts + (int64_t)row * a.n_parts;
        float m = ninf;
        for (int i = lane; i < a.n_parts; i += 64) m = fmaxf(m, pp[i].m);
        m = beam_wave_max(m);
        if (beam_finite(m)) {
          float s = 0.f;
          for (int i = lane; i < a.n_parts; i += 64) s += pp[i].sum * __expf(pp[i].m - m);
          s = beam_wave_sum(s);
          l = m + logf(s);
          st = 1u;
        }
      }
    }
    if (lane == 0) { lse[k] = l; state[k] = st; }
  }
  __syncthreads();
  // item i: place i % n_out of part (i / n_out) % n_parts of beam i / (n_out * n_parts);
  // a finished beam has one, in its first place
  const int per_beam = a.n_parts * a.n_out, total = a.K * per_beam;
  auto item = [&](int i) -> BeamCand {
    const int k = i / per_beam, r = i - k * per_beam;
    const uint32_t st = state[k];
    BeamCand x{0ull, 0ull};
    if (st == 0u) return x;
    const int row = row0 + k;
    float score;
    if (st == 2u) {
      if (r != 0) return x;
      score = a.scores[row];
      x.lo = 0xffffffffu - a.eos;
    } else {
      const int64_t slot = (int64_t)row * a.n_parts + r / a.n_out;
      if ((uint32_t)(r % a.n_out) >= a.parts[slot].n) return x;
      x.lo = a.cand[slot * a.n_out + r % a.n_out];
      score = a.scores[row] + (beam_okey_inv((uint32_t)(x.lo >> 32)) - lse[k]);
      if (!beam_finite(score)) return x;
    }
    x.hi = ((uint64_t)beam_okey(score) << 32) | (0xffffffffu - (uint32_t)k);
    return x;
  };
  uint32_t best[1] = {0u};
  for (int i = tid; i < total; i += kFinishThreads) best[0] = max(best[0], (uint32_t)(item(i).hi >> 32));
  const uint32_t bound = max(beam_bound<1, W>(best, a.n_out, red), 1u);
  for (int i = tid; i < total; i += kFinishThreads) {
    const BeamCand x = item(i);
    if ((uint32_t)(x.hi >> 32) >= bound) {
      const uint32_t o = atomicAdd(&counter, 1u);
      if (o < (uint32_t)kFinishSlots) slots[o] = x;
    }
  }
  __syncthreads();
  const int n = (int)counter;
  const int64_t o0 = (int64_t)b * a.n_out;
  auto put = [&](int r, const BeamCand& x) {
    const int k = (int)(0xffffffffu - (uint32_t)x.hi);
    const uint32_t tok = 0xffffffffu - (uint32_t)x.lo;
    a.out_scores[o0 + r] = beam_okey_inv((uint32_t)(x.hi >> 32));
    a.out_tokens[o0 + r] = tok;
    a.out_parents[o0 + r] = k;
    a.out_finished[o0 + r] = (state[k] == 2u || tok == a.eos) ? 1 : 0;
  };
  const int keep = min(n, a.n_out);
  for (int r = keep + tid; r < a.n_out; r += kFinishThreads) {  // places without a candidate
    a.out_scores[o0 + r] = ninf;
    a.out_tokens[o0 + r] = a.eos == HI_ROCM_BEAM_NO_EOS ? 0u : a.eos;
    a.out_parents[o0 + r] = r % a.K;
    a.out_finished[o0 + r] = 1;
  }
  if (n <= kFinishSlots) {
    if (tid < n) {
      const BeamCand mine = slots[tid];
      int rank = 0;
      for (int i = 0; i < n; ++i) rank += beam_before(slots[i], mine) ? 1 : 0;
      if (rank < a.n_out) put(rank, mine);
    }
    return;
  }
  // many equal scores: one candidate after another
  BeamCand prev{~0ull, ~0ull};
  for (int r = 0; r < keep; ++r) {
    BeamCand top{0ull, 0ull};
    for (int i = tid; i < total; i += kFinishThreads) {
      const BeamCand x = item(i);
      if (beam_before(prev, x) && beam_before(x, top)) top = x;
    }
    #pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      BeamCand w;
      w.hi = ((uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(top.hi >> 32), o, 64) << 32) |
             (uint32_t)__shfl_xor((int)(uint32_t)top.hi, o, 64);
      w.lo = ((uint64_t)(uint32_t)__shfl_xor((int)(uint32_t)(top.lo >> 32), o, 64) << 32) |
             (uint32_t)__shfl_xor((int)(uint32_t)top.lo, o, 64);
      if (beam_before(w, top)) top = w;
    }
    if (lane == 0) redc[wid] = top;
    __syncthreads();
    top = redc[0];
    #pragma unroll
    for (int w = 1; w < W; ++w)
      if (beam_before(redc[w], top)) top = redc[w];
    __syncthreads();
    prev = top;
    if (tid == 0) put(r, top);
  }
}

// Elements of a part: large parts once their workgroups fill the chip.
int beam_part_elems(int64_t rows, int V) {
  const int64_t large = rows * ((V + 7 + kPartThreads * 64 - 1) / (kPartThreads * 64));
  return kPartThreads * (large >= 512 ? 64 : 16);
}
int beam_parts(int64_t rows, int V) {
  const int e = beam_part_elems(rows, V);
  return (V + 7 + e - 1) / e;  // (up to 7 elements before the row's start)
}

struct BeamLayout {
  size_t cand, total;
};
BeamLayout beam_layout(int64_t slots, int n_out) {
  auto align = [](size_t x) { return (x + 255) & ~(size_t)255; };
  BeamLayout L;
  L.cand = align((size_t)slots * sizeof(BeamPart));
  L.total = L.cand + align((size_t)slots * n_out * sizeof(uint64_t));
  return L;
}

template <int DT>
void launch_part(const BeamArgs& a, int rows, int elems, hipStream_t st) {
  const dim3 grid((unsigned)a.n_parts, (unsigned)rows);
  if (elems == kPartThreads * 64) hipLaunchKernelGGL((beam_part_kernel<DT, 64>), grid, dim3(kPartThreads), 0, st, a);
  else hipLaunchKernelGGL((beam_part_kernel<DT, 16>), grid, dim3(kPartThreads), 0, st, a);
}

// ---- states ---------------------------------------------------------------

struct ReorderArgs {
  const char* src;
  char* dst;
  const int32_t* parents;  // [batch][K]
  const int32_t* lengths;  // [batch] or null
  int K;
  int64_t outer, mid, positions, pos_bytes;
  int64_t outer_stride, row_stride, mid_stride;
  int64_t cols;  // units of a row's piece: ceil(positions * pos_bytes / unit)
};

// One thread owns one unit (16, 4 or 1 bytes) of all K rows of a request: it
// reads what the rows need before it writes any of them, so dst may be src.
template <typename T, int KM>
__global__ void __launch_bounds__(256) beam_reorder_kernel(ReorderArgs a) {
  const int b = blockIdx.y;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.outer * a.mid * a.cols) return;
  const int64_t piece = i / a.cols, col = i - piece * a.cols;
  int64_t len = a.positions;
  if (a.lengths) {
    const int64_t l = a.lengths[b];
    len = l < 0 ? 0 : (l < len ? l : len);
  }
  if (col * (int64_t)sizeof(T) >= len * a.pos_bytes) return;
  const int64_t o = piece / a.mid, m = piece - o * a.mid;
  const int64_t at = o * a.outer_stride + m * a.mid_stride + (int64_t)b * a.K * a.row_stride + col * (int64_t)sizeof(T);
  const bool same = a.src == a.dst;
  T v[KM];
  int from[KM];
  #pragma unroll
  for (int j = 0; j < KM; ++j) {
    from[j] = -1;
    if (j < a.K) {
      const int p = a.parents[b * a.K + j];
      const int q = p < 0 || p >= a.K ? j : p;  // (a parent outside the request: the row stays)
      if (!same || q != j) {
        from[j] = q;
        v[j] = *reinterpret_cast<const T*>(a.src + at + q * a.row_stride);
      }
    }
  }
  #pragma unroll
  for (int j = 0; j < KM; ++j)
    if (from[j] >= 0) *reinterpret_cast<T*>(a.dst + at + j * a.row_stride) = v[j];
}

template <typename T>
void launch_reorder(ReorderArgs a, int batch, hipStream_t st) {
  a.cols = (a.positions * a.pos_bytes + (int64_t)sizeof(T) - 1) / (int64_t)sizeof(T);
  const dim3 grid((unsigned)((a.outer * a.mid * a.cols + 255) / 256), (unsigned)batch);
  if (a.K <= 4) hipLaunchKernelGGL((beam_reorder_kernel<T, 4>), grid, dim3(256), 0, st, a);
  else if (a.K <= 8) hipLaunchKernelGGL((beam_reorder_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else if (a.K <= 16) hipLaunchKernelGGL((beam_reorder_kernel<T, 16>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((beam_reorder_kernel<T, 32>), grid, dim3(256), 0, st, a);
}

}  // namespace
}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_beam_workspace_bytes(int max_batch, int beams, int vocab, int n_out, size_t* out_bytes) {
  if (max_batch <= 0 || beams <= 0 || vocab <= 0 || n_out <= 0 || out_bytes == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_workspace_bytes: invalid arguments");
  if (beams > kBeamMax || n_out > kBeamMaxOut || vocab > kMaxVocab || (int64_t)max_batch * beams > kBeamMaxRows)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_beam_workspace_bytes: more than 32 beams, 64 outputs, 65536 rows or 2^23 tokens");
  int64_t slots = 0;
  for (int b = 1; b <= max_batch; ++b)
    slots = std::max(slots, (int64_t)b * beams * beam_parts((int64_t)b * beams, vocab));
  *out_bytes = beam_layout(slots, n_out).total;
  return HI_ROCM_OK;
}

int hi_rocm_beam_select(const void* logits, int dtype, int batch, int beams, int vocab, int64_t row_stride,
                        const float* scores, const uint8_t* finished, uint32_t eos_id, const uint32_t* mask_words,
                        int n_out, float* out_scores, uint32_t* out_tokens, int32_t* out_parents,
                        uint8_t* out_finished, void* workspace, size_t workspace_bytes, void* stream) {
  if (logits == nullptr || scores == nullptr || out_scores == nullptr || out_tokens == nullptr ||
      out_parents == nullptr || out_finished == nullptr || batch <= 0 || beams <= 0 || vocab <= 0 || n_out <= 0 ||
      row_stride < vocab)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_select: invalid arguments");
  if (dtype != HI_ROCM_DTYPE_F32 && dtype != HI_ROCM_DTYPE_BF16)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_select: unknown dtype");
  if ((uintptr_t)logits % (dtype == HI_ROCM_DTYPE_F32 ? 4 : 2) != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_select: logits not aligned to their type");
  if (finished != nullptr && eos_id == HI_ROCM_BEAM_NO_EOS)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_select: finished beams need an eos id");
  if (beams > kBeamMax || n_out > kBeamMaxOut || vocab > kMaxVocab || (int64_t)batch * beams > kBeamMaxRows - 1)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_beam_select: more than 32 beams, 64 outputs, 65535 rows or 2^23 tokens");
  const int rows = batch * beams;
  BeamArgs a;
  memset(&a, 0, sizeof(a));
  a.n_parts = beam_parts(rows, vocab);
  const BeamLayout L = beam_layout((int64_t)rows * a.n_parts, n_out);
  if (workspace == nullptr || workspace_bytes < L.total || (uintptr_t)workspace % 16 != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_select: workspace missing, too small or not 16-byte aligned");
  a.logits = logits;
  a.row_stride = row_stride;
  a.scores = scores;
  a.finished = finished;
  a.mask = mask_words;
  a.V = vocab;
  a.K = beams;
  a.n_out = n_out;
  a.mask_words = (vocab + 31) / 32;
  a.eos = eos_id;
  a.parts = (BeamPart*)workspace;
  a.cand = (uint64_t*)((char*)workspace + L.cand);
  a.out_scores = out_scores;
  a.out_tokens = out_tokens;
  a.out_parents = out_parents;
  a.out_finished = out_finished;
  const int elems = beam_part_elems(rows, vocab);
  if (dtype == HI_ROCM_DTYPE_F32) launch_part<HI_ROCM_DTYPE_F32>(a, rows, elems, (hipStream_t)stream);
  else launch_part<HI_ROCM_DTYPE_BF16>(a, rows, elems, (hipStream_t)stream);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return api_hip_fail(e, "beam part launch");
  hipLaunchKernelGGL(beam_finish_kernel, dim3((unsigned)batch), dim3(kFinishThreads), 0, (hipStream_t)stream, a);
  e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "beam finish launch");
}

int hi_rocm_beam_reorder(const void* src, void* dst, const int32_t* parents, int batch, int beams, int64_t outer,
                         int64_t outer_stride, int64_t row_stride, int64_t mid, int64_t mid_stride, int64_t positions,
                         int64_t pos_bytes, const int32_t* lengths, void* stream) {
  if (src == nullptr || dst == nullptr || parents == nullptr || batch <= 0 || beams <= 0 || outer <= 0 || mid <= 0 ||
      positions <= 0 || pos_bytes <= 0 || outer_stride < 0 || row_stride < 0 || mid_stride < 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_reorder: invalid arguments");
  if (beams > kBeamMax || batch > kBeamMaxRows - 1)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_beam_reorder: more than 32 beams or 65535 requests");
  constexpr int64_t kBig = (int64_t)1 << 46;
  if (positions > kBig / pos_bytes || outer > kBig || mid > kBig || outer_stride > kBig || row_stride > kBig ||
      mid_stride > kBig)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_beam_reorder: sizes above 2^46 bytes");
  // pieces of different rows, outer and mid indexes must not share bytes:
  // from the smallest stride up, each at least what lies inside it
  const int64_t rows = (int64_t)batch * beams, piece = positions * pos_bytes;
  struct Dim { int64_t stride, n; } d[3] = {{outer_stride, outer}, {row_stride, rows}, {mid_stride, mid}};
  std::sort(d, d + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
  int64_t extent = piece;
  for (const Dim& x : d) {
    if (x.n == 1) continue;
    if (x.stride < extent)
      return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_reorder: strides let rows overlap");
    if (x.n - 1 > (kBig - extent) / x.stride)
      return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_beam_reorder: sizes above 2^46 bytes");
    extent += (x.n - 1) * x.stride;
  }
  const uintptr_t s = (uintptr_t)src, t = (uintptr_t)dst;
  if (s != t && s < t + (uintptr_t)extent && t < s + (uintptr_t)extent)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_beam_reorder: src and dst overlap without being the same");
  ReorderArgs a;
  memset(&a, 0, sizeof(a));
  a.src = (const char*)src;
  a.dst = (char*)dst;
  a.parents = parents;
  a.lengths = lengths;
  a.K = beams;
  a.outer = outer;
  a.mid = mid;
  a.positions = positions;
  a.pos_bytes = pos_bytes;
  a.outer_stride = outer > 1 ? outer_stride : 0;
  a.row_stride = rows > 1 ? row_stride : 0;
  a.mid_stride = mid > 1 ? mid_stride : 0;
  const uint64_t bits = s | t | (uint64_t)a.outer_stride | (uint64_t)a.row_stride | (uint64_t)a.mid_stride |
                        (uint64_t)pos_bytes;
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  if ((outer * mid * ((piece + unit - 1) / unit) + 255) / 256 > INT32_MAX)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_beam_reorder: more than 2^39 units a request");
  if (unit == 16) launch_reorder<int4>(a, batch, (hipStream_t)stream);
  else if (unit == 4) launch_reorder<uint32_t>(a, batch, (hipStream_t)stream);
  else launch_reorder<uint8_t>(a, batch, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "beam reorder launch");
}

}  // extern "C"
