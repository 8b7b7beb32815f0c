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
// Two kernels, the first reads each logit once:
//  * a part of a row: its maximum, its sum of exponentials, and its first n_out
//    candidates by (logit, token); beam_tile_kernel while the parts are few,
//    beam_part_kernel for many rows;
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
constexpr int kTileElems = 4096;     // elements of a part of a short step
constexpr int kTileSlots = 512;      // candidates that such a part can hold before it ranks them
constexpr int kPartSlots = 256;      // groups of four logits that a wave of a streamed part can hold
constexpr int kFinishThreads = 512;
constexpr int kFinishHeld = 4;       // candidates a thread keeps in registers
constexpr int kFinishSlots = 512;
constexpr int kBeamMaxRows = 65535;  // (a grid's second dimension)

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
  int tiles;                  // of a part
  int list_threads;           // log2 of the threads that take a part's list in the finish
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
constexpr float kBeamLog2e = 1.44269502e+00f;
constexpr float kBeamFused = 1e30f;  // logits up to this size can be scaled by log2 e
constexpr float kBeamLowest = -3.402823466e38f;
constexpr uint32_t kBeamNegInf = 0x007fffffu;  // beam_okey(-inf): keys above it are candidates

// The largest of three numbers.  (fmaxf would first quiet each operand, an
// instruction a logit.)  A quiet NaN is passed over, but a signalling one takes
// the place of all before it: whoever may have met a NaN, which shows in the sum
// of the exponentials, takes NaN out and the maxima again.
__device__ __forceinline__ float beam_max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

// Wave reductions by DPP moves (lane 63 ends with the result).
template <typename F>
__device__ __forceinline__ uint32_t beam_wave_fold(uint32_t v, F f) {
  v = f(v, dpp32<kDppShr1>(v, v));
  v = f(v, dpp32<kDppShr1 + 1>(v, v));
  v = f(v, dpp32<kDppShr1 + 3>(v, v));
  v = f(v, dpp32<kDppShr1 + 7>(v, v));
  v = f(v, dpp32<kDppBcast15, 0xa>(v, v));
  v = f(v, dpp32<kDppBcast31, 0xc>(v, v));
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t beam_wave_umax(uint32_t v) {
  return beam_wave_fold(v, [](uint32_t x, uint32_t y) { return max(x, y); });
}
__device__ __forceinline__ uint32_t beam_wave_umin(uint32_t v) {
  return beam_wave_fold(v, [](uint32_t x, uint32_t y) { return min(x, y); });
}
__device__ __forceinline__ float beam_wave_max(float v) {
  return __uint_as_float(beam_wave_fold(__float_as_uint(v), [](uint32_t x, uint32_t y) {
    return __float_as_uint(beam_max3(__uint_as_float(x), __uint_as_float(y), __uint_as_float(y)));
  }));
}
__device__ __forceinline__ float beam_wave_sum(float v) {
  auto add = [&](uint32_t w) { v += __uint_as_float(w); };
  auto b = [&]() { return __float_as_uint(v); };
  add(dpp32<kDppShr1, 0xf, true>(0u, b()));
  add(dpp32<kDppShr1 + 1, 0xf, true>(0u, b()));
  add(dpp32<kDppShr1 + 3, 0xf, true>(0u, b()));
  add(dpp32<kDppShr1 + 7, 0xf, true>(0u, b()));
  add(dpp32<kDppBcast15, 0xa>(0u, b()));
  add(dpp32<kDppBcast31, 0xc>(0u, b()));
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)b(), 63));
}

// The sum over a lane's eight neighbours 8 i .. 8 i + 7.
__device__ __forceinline__ int beam_sum8(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xf, 0xf, true);   // lanes 1, 0, 3, 2
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xf, 0xf, true);   // lanes 2, 3, 0, 1
  return v + __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, true);  // mirrored within the eight
}

// N elements that are tokens t .. t + N - 1, where they are outside the row or
// masked: -inf.  lo and hi: the mask word of max(t, 0) and the next one (~0: none).
template <int N>
__device__ __forceinline__ void beam_leave_out(float* x, int t, int V, uint32_t lo, uint32_t hi) {
  uint32_t bits = (uint32_t)(((uint64_t)hi << 32 | lo) >> (max(t, 0) & 31));
  if (t < 0) bits <<= -t;
  bits &= (1u << min(max(V - t, 0), N)) - 1u;
  #pragma unroll
  for (int q = 0; q < N; ++q) {
    const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)bits, q, 1);
    x[q] = __uint_as_float((__float_as_uint(x[q]) & keep) | (0xff800000u & ~keep));
  }
}

// Whether a row takes part: a beam whose score is not finite has no
// candidates, a finished one has a single candidate that needs no logits.
struct BeamFlag {  // (its loads go out where it is made; without flags it reads a byte of the score)
  float score;
  bool flags;
  uint8_t done;
  __device__ __forceinline__ BeamFlag(const BeamArgs& a, int row)
      : score(a.scores[row]), flags(a.finished != nullptr),
        done(*(flags ? a.finished + row : reinterpret_cast<const uint8_t*>(a.scores + row))) {}
  __device__ __forceinline__ bool finished() const {
    uint32_t d = done;
    asm volatile("" : "+v"(d));  // (looked at here, not where it was loaded)
    return flags && d != 0u;
  }
  __device__ __forceinline__ bool reads() const { return beam_finite(score) && !finished(); }
};

// A key that at least n <= 64 of G keys a lane reach, and not many more: from
// the bits that the largest key and the smallest lane's largest (64 keys reach
// it) share downwards, until at most n + n / 2 + 1 reach it.
template <int G>
__device__ __forceinline__ uint32_t beam_wave_nth(const uint32_t (&key)[G], int n) {
  uint32_t top = key[0];
  #pragma unroll
  for (int g = 1; g < G; ++g) top = max(top, key[g]);
  const uint32_t hi = beam_wave_umax(top);
  if (n == 1) return hi;
  const uint32_t lo = beam_wave_umin(top);
  if (lo == hi) return lo;
  const int first = 31 - __builtin_clz(lo ^ hi);
  uint32_t t = hi & ~((2u << first) - 1u);
  #pragma unroll 1
  for (int bit = first; bit >= 0; --bit) {
    const uint32_t c = t | (1u << bit);
    int cnt = 0;
    #pragma unroll
    for (int g = 0; g < G; ++g) cnt += __popcll(__ballot(key[g] >= c));
    if (cnt >= n) {
      t = c;
      if (cnt <= n + n / 2 + 1) break;
    }
  }
  return t;
}

// A bound that at least n keys of the workgroup (W waves, G keys a lane)
// reach, if it holds n above `floor`: the smallest of the waves' ceil(n /
// W)-th keys, or, where a wave has not as many (a row's last part), the m-th
// largest of their ceil(n / m)-th, m = W / 2, W / 4, ..., 1.
template <int G, int W>
__device__ __forceinline__ uint32_t beam_bound(const uint32_t (&key)[G], int n, uint32_t floor, uint32_t* red) {
  const int wid = threadIdx.x >> 6;
  const uint32_t share = beam_wave_nth<G>(key, (n + W - 1) / W);
  if ((threadIdx.x & 63) == 0) red[wid] = share;
  __syncthreads();
  uint32_t b = red[0];
  #pragma unroll
  for (int w = 1; w < W; ++w) b = min(b, red[w]);
  int had = (n + W - 1) / W;
  #pragma unroll 1
  for (int m = W / 2; m >= 1 && b <= floor; m /= 2) {
    uint32_t mine = red[threadIdx.x & (W - 1)];  // (lane w < W: wave w's)
    // (waves without as many keys have no more)
    if (__popcll(__ballot(mine > floor) & ((1ull << W) - 1ull)) < m) continue;
    const int need = (n + m - 1) / m;
    if (need != had) {
      const uint32_t more = beam_wave_nth<G>(key, need);
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[wid] = more;
      __syncthreads();
      had = need;
      mine = red[threadIdx.x & (W - 1)];
    }
    #pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)mine, w);
      if (__popcll(__ballot(mine >= r) & ((1ull << W) - 1ull)) >= m) b = max(b, r);
    }
  }
  return b;
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

// One part of a short step: kTileElems elements of a row, counted from the
// 16-byte boundary at or before the row's start (rows start anywhere; the
// elements before the start and after the end are no candidates).  All of it
// is in registers at once, and little code runs, which is most of such a
// launch's time: 4 rows of 151,936 f32 take 6.0 us, 8.2 with the streaming
// kernel below; 120 masked rows of 50,257 (1,560 parts) 10 us.
template <int DT>
__global__ void __launch_bounds__(kPartThreads) beam_tile_kernel(BeamArgs a) {
  constexpr int PER = kTileElems / kPartThreads;
  constexpr int N = BeamLoad<DT>::N, L = PER / N, W = kPartThreads / 64, ES = 16 / N;
  constexpr int G = PER / 8;  // groups a thread
  __shared__ uint64_t slots[kTileSlots];
  __shared__ uint64_t red64[W];
  __shared__ uint32_t red[W];
  __shared__ float redf[W], reds[W];
  __shared__ uint32_t counter;
  const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const char* p0 = (const char*)a.logits + (int64_t)row * a.row_stride * ES;
  const int head = (int)((uintptr_t)p0 & 15) / ES;
  const int64_t base = (int64_t)part * (kPartThreads * PER);  // elements from the aligned start
  // range-checked loads: bytes from this part's start to the row's end
  const int64_t left = ((int64_t)a.V + head - base) * ES;  // (the last part may lie after the row: nothing)
  constexpr int64_t kSpan = (int64_t)kPartThreads * PER * ES;
  const int bytes = left < 0 ? 0 : (int)(left < kSpan ? left : kSpan);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p0 - head * ES + base * ES), 0, (bytes + 3) & ~3, kBufferConfig);
  if (tid == 0) counter = 0u;
  const float ninf = -__builtin_inff();
  // token of x[j * N + q]: t0 + j * kPartThreads * N + q
  const int t0 = (int)base + tid * N - head;
  // Inside the row and without a mask nothing is left out but NaN, which shows
  // in the sum.
  const bool inside = base >= head && base - head + kPartThreads * PER <= a.V && a.mask == nullptr;
  const uint32_t* mrow = a.mask ? a.mask + (int64_t)row * a.mask_words : nullptr;
  // all loads go out before it is known that the row takes part
  const BeamFlag flag(a, row);
  i32x4_t v[L];
  #pragma unroll
  for (int j = 0; j < L; ++j) v[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, (j * kPartThreads + tid) * 16, 0, 0);
  uint32_t lo[L], hi[L];
  #pragma unroll
  for (int j = 0; j < L; ++j) lo[j] = hi[j] = ~0u;
  if (mrow) {
    #pragma unroll
    for (int j = 0; j < L; ++j) {
      const int w = min(max(t0 + j * (kPartThreads * N), 0) >> 5, a.mask_words - 1);
      lo[j] = mrow[w];
      hi[j] = mrow[min(w + 1, a.mask_words - 1)];  // (unused where N tokens from a multiple of N share a word)
    }
  }
  if (!flag.reads()) return;
  float x[PER];
  #pragma unroll
  for (int j = 0; j < L; ++j) {
    #pragma unroll
    for (int q = 0; q < N; ++q) x[j * N + q] = BeamLoad<DT>::get(v[j], q);
  }
  if (!inside) {
    #pragma unroll
    for (int j = 0; j < L; ++j) beam_leave_out<N>(x + j * N, t0 + j * (kPartThreads * N), a.V, lo[j], hi[j]);
  }
  float gm[G], m;
  auto maxima = [&]() {
    #pragma unroll
    for (int g = 0; g < G; ++g) {
      gm[g] = ninf;
      #pragma unroll
      for (int i = 0; i < 8; i += 2) gm[g] = beam_max3(gm[g], x[8 * g + i], x[8 * g + i + 1]);
    }
    static_assert(G == 2, "two groups a thread");
    m = beam_wave_max(beam_max3(gm[0], gm[1], ninf));
  };
  maxima();
  // each wave's sum by its own maximum, so that one exchange serves both
  float s = 0.f;
  bool odd = !beam_finite(m) || fabsf(m) > kBeamFused;  // (products that overflow)
  if (!odd) {
    // e^(x - m) as 2^(x log2 e - m log2 e), as in the streaming kernel below
    const float shift = -m * kBeamLog2e;
    #pragma unroll
    for (int i = 0; i < PER; ++i) s += __builtin_amdgcn_exp2f(fmaf(x[i], kBeamLog2e, shift));
    odd = __ballot(!(s == s)) != 0ull;  // a NaN logit
  }
  if (odd) {
    // (a signalling NaN may have replaced the maxima found before it, the wave's
    // among them)
    #pragma unroll
    for (int i = 0; i < PER; ++i) x[i] = x[i] == x[i] ? x[i] : ninf;
    maxima();
    s = 0.f;
    if (beam_finite(m)) {
      #pragma unroll
      for (int i = 0; i < PER; ++i) s += __expf(x[i] - m);
    }
  }
  s = beam_wave_sum(s);
  if (lane == 0) { redf[wid] = m; reds[wid] = s; }
  // the part's candidates: all logits at or above a bound that n_out of them reach
  uint32_t key[G];
  #pragma unroll
  for (int g = 0; g < G; ++g) key[g] = beam_okey(gm[g]);
  const uint32_t bound = max(beam_bound<G, W>(key, a.n_out, kBeamNegInf, red), kBeamNegInf + 1u);
  m = redf[0];
  #pragma unroll
  for (int w = 1; w < W; ++w) m = fmaxf(m, redf[w]);
  const int64_t slot = (int64_t)row * a.n_parts + part;
  if (!beam_finite(m)) {  // nothing allowed, or a +inf logit: the finish sees which
    if (tid == 0) a.parts[slot] = BeamPart{m, 0.f, 0u, 0u};
    return;
  }
  const float at_least = beam_okey_inv(bound);
  #pragma unroll
  for (int g = 0; g < G; ++g) {
    if (gm[g] < at_least) continue;
    #pragma unroll
    for (int i = 8 * g; i < 8 * g + 8; ++i) {
      if (x[i] >= at_least) {
        const uint32_t o = atomicAdd(&counter, 1u);
        const int t = t0 + i / N * (kPartThreads * N) + i % N;
        if (o < (uint32_t)kTileSlots) slots[o] = ((uint64_t)beam_okey(x[i]) << 32) | (0xffffffffu - (uint32_t)t);
      }
    }
  }
  __syncthreads();
  int n = (int)counter;
  uint64_t* out = a.cand + slot * a.n_out;
  const int keep = min(n, a.n_out);
  if (tid == 0) {
    s = 0.f;
    #pragma unroll
    for (int w = 0; w < W; ++w) s += reds[w] * __expf(redf[w] - m);
    a.parts[slot] = BeamPart{m, s, (uint32_t)keep, 0u};
  }
  if (n <= kTileSlots) {
    // far more than n_out (a row's last part): only those that reach a better bound
    if (n > 2 * a.n_out + 64) {
      static_assert(kTileSlots == 2 * kPartThreads, "two slots a thread");
      const uint64_t own[2] = {tid < n ? slots[tid] : 0ull, tid + kPartThreads < n ? slots[tid + kPartThreads] : 0ull};
      const uint32_t half[2] = {(uint32_t)(own[0] >> 32), (uint32_t)(own[1] >> 32)};
      const uint32_t least = beam_bound<2, W>(half, a.n_out, 0u, red);
      __syncthreads();
      if (tid == 0) counter = 0u;
      __syncthreads();
      #pragma unroll
      for (int j = 0; j < 2; ++j)
        if (half[j] >= least) slots[atomicAdd(&counter, 1u)] = own[j];
      __syncthreads();
      n = (int)counter;
    }
    // ranks by counting, eight lanes a candidate
    for (int j = tid >> 3; j < n; j += kPartThreads / 8) {
      const uint64_t mine = slots[j];
      int rank = 0;
      #pragma unroll 4
      for (int i = tid & 7; i < n; i += 8) rank += slots[i] > mine;
      rank = beam_sum8(rank);
      if ((tid & 7) == 0 && rank < a.n_out) out[rank] = mine;
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
        if (x[j * N + q] >= at_least && k < prev && k > best) best = k;
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

// Groups of four neighbouring logits, as a wave of a streamed part lists them.
typedef float beam_f32x4 __attribute__((ext_vector_type(4)));
struct BeamList {
  beam_f32x4 x[kPartSlots];
  uint32_t token[kPartSlots];  // of the first
};
// Set bits of a ballot below this lane's.
__device__ __forceinline__ int beam_below(uint64_t b) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0u));
}
// The keys of group i's logits (0: below `floor`, or not in the list).
__device__ __forceinline__ void beam_keys(const BeamList* list, int i, int count, uint32_t floor, uint64_t (&k)[4]) {
  const beam_f32x4 x = list->x[min(i, kPartSlots - 1)];
  const uint32_t t = list->token[min(i, kPartSlots - 1)];
  #pragma unroll
  for (int q = 0; q < 4; ++q) {
    const uint32_t o = beam_okey(x[q]);
    k[q] = i < count && o >= floor ? (uint64_t)o << 32 | (0xffffffffu - (t + q)) : 0ull;
  }
}

// The keys (logit, token) of the first n of a list's logits whose ordered bits
// reach `floor`, in any order; returns how many.  A threshold is found bit by
// bit from the highest bit in which the keys differ.  ONE: at most 64 groups,
// whose keys stay in registers; else every step takes them from the list again.
template <bool ONE>
__device__ __forceinline__ int beam_first(const BeamList* list, int count, int n, uint32_t floor, uint64_t* out) {
  const int lane = threadIdx.x & 63;
  uint64_t k[4];
  uint32_t hi = 0u, lo = 0xffffffffu;  // of the keys' upper halves
  int all = 0;
  #pragma unroll 1
  for (int i = 0; i < (ONE ? 1 : count); i += 64) {
    beam_keys(list, i + lane, count, floor, k);
    #pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t o = (uint32_t)(k[q] >> 32);
      hi = max(hi, o);
      lo = min(lo, o - 1u);  // (0: none)
      all += __popcll(__ballot(o != 0u));
    }
  }
  uint64_t t = 1ull;
  if (all > n) {
    hi = beam_wave_umax(hi);
    lo = beam_wave_umin(lo) + 1u;
    int bit = hi == lo ? 31 : 63 - __builtin_clz(hi ^ lo);
    t = (uint64_t)hi << 32 & ~((2ull << bit) - 1ull);
    #pragma unroll 1
    for (; bit >= 0; --bit) {
      const uint64_t c = t | (1ull << bit);
      int cnt = 0;
      #pragma unroll 1
      for (int i = 0; i < (ONE ? 1 : count); i += 64) {
        if (!ONE) beam_keys(list, i + lane, count, floor, k);
        #pragma unroll
        for (int q = 0; q < 4; ++q) cnt += __popcll(__ballot(k[q] >= c));
      }
      if (cnt >= n) t = c;
      if (cnt == n) break;
    }
  }
  int at = 0;
  #pragma unroll 1
  for (int i = 0; i < (ONE ? 1 : count); i += 64) {
    if (!ONE) beam_keys(list, i + lane, count, floor, k);
    #pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint64_t keep = __ballot(k[q] >= t);
      if (k[q] >= t) out[at + beam_below(keep)] = k[q];
      at += __popcll(keep);
    }
  }
  return at;
}
// (Not inlined: the loop over a part has a place for it a group.)
__device__ __noinline__ int beam_first_of_many(const BeamList* list, int count, int n, uint32_t floor, uint64_t* out) {
  return beam_first<false>(list, count, n, floor, out);
}

// One part of a row: tiles [part * a.tiles, ...) of 64 lanes x 64 bytes,
// counted from the 16-byte boundary at or before the row's start (rows start
// anywhere; what lies before the start and after the end is no candidate).
// Each wave takes every fourth tile, with the next one's loads in flight, and
// needs no other wave until the end:
//  * a lane keeps its running maximum and sum, rescaled once a tile;
//  * the wave keeps its candidates in LDS, as groups of four logits that hold
//    one at or above a bound: one that n_out of the four first tiles' groups
//    reach, or the n_out-th kept after a full list was cut back to n_out, so
//    that most tiles end at one comparison.
// Parts of kTileElems by the kernel above instead have more instructions a logit
// and no loads in flight while they compute (64 x 8 rows of 151,936 bf16, a
// fifth of them finished, the whole step: 57 us, with this kernel 41).  What
// bounds it: bytes behind 64 MB (6.3 TB/s from 65,536 to 262,144 logits a row),
// and about 16 us of launches, first and last tiles, and the finish.
template <int DT, bool MASK>
__global__ void __launch_bounds__(kPartThreads) beam_part_kernel(BeamArgs a) {
  constexpr int N = BeamLoad<DT>::N, L = 4, PER = L * N, W = kPartThreads / 64, ES = 16 / N;
  constexpr int G = PER / 4, GN = 4;  // groups of 4 elements
  __shared__ BeamList lists[W];
  __shared__ uint64_t keys[W][kBeamMaxOut];
  __shared__ float redm[W], reds[W];
  __shared__ int redn[W];
  __shared__ uint32_t red[W];
  // what a wave's share of n_out lanes reach (0: nothing yet); not `red`, which a
  // slower wave may still read when a faster one is a tile ahead
  __shared__ uint32_t reach[W];
  const int row = blockIdx.y, part = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const char* p0 = (const char*)a.logits + (int64_t)row * a.row_stride * ES;
  const int head = (int)((uintptr_t)p0 & 15) / ES;
  // range-checked loads: bytes from this part's start to the row's or its end
  const int64_t base = (int64_t)part * a.tiles * (64 * PER);  // elements from the aligned start
  const int64_t left = ((int64_t)a.V + head - base) * ES;     // (the last part may lie after the row: nothing)
  const int64_t span = (int64_t)a.tiles * (64 * 16 * L);
  const int bytes = left < 0 ? 0 : (int)(left < span ? left : span);
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
      (void*)(p0 - head * ES + base * ES), 0, (bytes + 3) & ~3, kBufferConfig);
  const uint32_t* mrow = MASK ? a.mask + (int64_t)row * a.mask_words : nullptr;
  i32x4_t next[L];
  uint32_t word[L], word2[L];  // the mask words of the first token of each load and the next one
  auto load = [&](int tile) {
    #pragma unroll
    for (int j = 0; j < L; ++j)
      next[j] = __builtin_amdgcn_raw_buffer_load_b128(rs, tile * (64 * 16 * L) + (j * 64 + lane) * 16, 0, 0);
    if (MASK) {
      const int64_t t = base + (int64_t)tile * (64 * PER) - head + lane * N;
      #pragma unroll
      for (int j = 0; j < L; ++j) {
        const int w = (int)min(max(t + j * (64 * N), (int64_t)0) >> 5, (int64_t)a.mask_words - 1);
        word[j] = mrow[w];
        word2[j] = head != 0 ? mrow[min(w + 1, a.mask_words - 1)] : ~0u;  // (N tokens from a multiple of N share a word)
      }
    }
  };
  // (the first loads go out before it is known that the row takes part)
  const BeamFlag flag(a, row);
  load(wid);
  if (!flag.reads()) return;
  const float ninf = -__builtin_inff();
  BeamList* list = &lists[wid];
  int count = 0, since = 0;    // groups in it, and those listed since the bound rose
  float m = ninf, s = 0.f;     // this lane's
  float bound = 0.f;           // candidates are at or above it; once `full`, above it in the next tile
  bool full = false, shared = false;
  auto shared_bound = [&]() {
    const uint32_t key[1] = {beam_okey(m)};
    volatile uint32_t* v = reach;
    const uint32_t own = beam_wave_nth<1>(key, (a.n_out + W - 1) / W);
    if (lane == 0) v[wid] = own;
    uint32_t b = own;
    #pragma unroll
    for (int w = 0; w < W; ++w) b = min(b, v[w]);
    return (uint32_t)__builtin_amdgcn_readfirstlane((int)b);
  };
  for (int tile = wid; tile < a.tiles; tile += W) {
    float x[PER];
    #pragma unroll
    for (int j = 0; j < L; ++j) {
      #pragma unroll
      for (int q = 0; q < N; ++q) x[j * N + q] = BeamLoad<DT>::get(next[j], q);
    }
    uint32_t lo[L], hi[L];
    if (MASK) {
      #pragma unroll
      for (int j = 0; j < L; ++j) { lo[j] = word[j]; hi[j] = word2[j]; }
    }
    if (tile + W < a.tiles) load(tile + W);
    // token of x[j * N + q]: t0 + j * 64 * N + q
    const int64_t e0 = base + (int64_t)tile * (64 * PER) - head;
    if (e0 >= a.V && tile >= W) break;
    const int t0 = (int)e0 + lane * N;
    // Inside the row and without a mask nothing is left out but NaN, which shows
    // in the sum.
    if (e0 < 0 || e0 + 64 * PER > a.V || MASK) {
      #pragma unroll
      for (int j = 0; j < L; ++j)
        beam_leave_out<N>(x + j * N, t0 + j * (64 * N), a.V, MASK ? lo[j] : ~0u, MASK ? hi[j] : ~0u);
    }
    // the groups' maxima, and the sum about the running maximum (of a lane
    // without a logit: about a low value, which leaves its terms 0)
    float gm[G], tm, mn, at, add = 0.f;
    auto maxima = [&]() {
      #pragma unroll
      for (int g = 0; g < G; ++g)
        gm[g] = beam_max3(beam_max3(x[GN * g], x[GN * g + 1], x[GN * g + 2]), x[GN * g + 3], ninf);
      tm = gm[0];
      #pragma unroll
      for (int g = 1; g + 1 < G; g += 2) tm = beam_max3(tm, gm[g], gm[g + 1]);
      tm = beam_max3(tm, gm[G - 1], ninf);
      mn = beam_max3(m, tm, ninf);
    };
    maxima();
    // e^(x - at) as 2^(x log2 e - at log2 e), one fused operation and the
    // exponential: the second product's rounding is that of a number of at's
    // size, as the rounding of lse will be.
    at = beam_max3(mn, -kBeamFused, ninf);
    const float shift = -at * kBeamLog2e;
    #pragma unroll
    for (int i = 0; i < PER; ++i) add += __builtin_amdgcn_exp2f(fmaf(x[i], kBeamLog2e, shift));
    // NaN logits (masked; +inf: the sum does not matter) and logits whose
    // products overflow
    const bool odd = !(add < __builtin_inff()) || mn > kBeamFused || (mn < -kBeamFused && mn > ninf);
    if (__ballot(odd) != 0ull) {
      #pragma unroll
      for (int i = 0; i < PER; ++i) x[i] = x[i] == x[i] ? x[i] : ninf;
      maxima();
      at = beam_max3(mn, kBeamLowest, ninf);
      add = 0.f;
      #pragma unroll
      for (int i = 0; i < PER; ++i) add += __expf(x[i] - at);
    }
    s = s * __expf(beam_max3(m, kBeamLowest, ninf) - at) + add;
    m = mn;
    // candidates
    if (tile < W) {  // every wave's first
      uint32_t key[G / 2];  // groups of 8
      #pragma unroll
      for (int g = 0; g < G / 2; ++g) key[g] = beam_okey(beam_max3(gm[2 * g], gm[2 * g + 1], ninf));
      if (lane == 0) reach[wid] = 0u;
      const uint32_t k = beam_bound<G / 2, W>(key, a.n_out, kBeamNegInf, red);
      shared = k > kBeamNegInf;
      bound = beam_okey_inv(max(k, kBeamNegInf + 1u));
    }
    // n_out kept, by this wave or in all first tiles: equal logits of later
    // tiles have higher tokens
    if (tile / W == 1 && shared) full = true;
    // The bound rises with what the waves have seen, after 2, 4, 8, ... tiles:
    // each keeps the value that its share of n_out lanes reach, and all values
    // at or above the least of these include n_out.  (One read early only
    // bounds less.  The others may be tiles ahead, so an equal logit may still
    // have a lower token.)
    if (tile >= W && (tile / W & (tile / W - 1)) == 0) {
      const float b = beam_okey_inv(shared_bound());
      if (b > bound) {
        bound = b;
        full = false;
        since = 0;
      }
    }
    const uint64_t any = __ballot(full ? tm > bound : tm >= bound);
    if (any == 0ull) continue;
    #pragma unroll
    for (int g = 0; g < G; ++g) {
      const bool pass = full ? gm[g] > bound : gm[g] >= bound;
      const uint64_t b = __ballot(pass);
      if (b == 0ull) continue;
      if (pass) {
        const int i = count + beam_below(b);
        list->x[i] = beam_f32x4{x[GN * g], x[GN * g + 1], x[GN * g + 2], x[GN * g + 3]};
        list->token[i] = (uint32_t)(t0 + GN * g / N * (64 * N) + GN * g % N);
      }
      count = __builtin_amdgcn_readfirstlane(count + __popcll(b));
      since = __builtin_amdgcn_readfirstlane(since + __popcll(b));
      if (count > kPartSlots - 64) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        count = __builtin_amdgcn_readfirstlane(
            beam_first_of_many(list, count, a.n_out, kBeamNegInf + 1u, keys[wid]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint32_t low = 0xffffffffu;
        if (lane < count) {
          const uint64_t k = keys[wid][lane];
          low = (uint32_t)(k >> 32);
          list->x[lane] = beam_f32x4{beam_okey_inv(low), ninf, ninf, ninf};
          list->token[lane] = 0xffffffffu - (uint32_t)k;
        }
        const float least = beam_okey_inv(beam_wave_umin(low));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // a later logit of this tile may equal it with a lower token
        if (least > bound) { bound = least; full = false; }
        // (after a rise by what other waves have seen, some kept are below it)
        since = __popcll(__ballot(lane < count && low >= beam_okey(bound)));
      }
    }
    if (since >= a.n_out) full = true;
  }
  if (a.tiles > W) shared_bound();
  {
    const float wm = beam_wave_max(m), at = fmaxf(wm, kBeamLowest);
    s = beam_wave_sum(s * __expf(fmaxf(m, kBeamLowest) - at));
    if (lane == 0) { redm[wid] = wm; reds[wid] = s; }
  }
  __syncthreads();
  m = redm[0];
  uint32_t last = reach[0];  // n_out of the part's logits reach it
  #pragma unroll
  for (int w = 1; w < W; ++w) {
    m = fmaxf(m, redm[w]);
    last = min(last, reach[w]);
  }
  const int64_t slot = (int64_t)row * a.n_parts + part;
  if (!beam_finite(m)) {  // nothing allowed, or a +inf logit: the finish sees which
    if (tid == 0) a.parts[slot] = BeamPart{m, 0.f, 0u, 0u};
    return;
  }
  if (tid == 0) {
    s = 0.f;
    #pragma unroll
    for (int w = 0; w < W; ++w) s += reds[w] * __expf(fmaxf(redm[w], kBeamLowest) - m);
  }
  // the wave's first n_out that reach it
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const uint32_t floor = a.tiles > W ? max(last, kBeamNegInf + 1u) : kBeamNegInf + 1u;
  if (count > 64)
    count = __builtin_amdgcn_readfirstlane(beam_first_of_many(list, count, a.n_out, floor, keys[wid]));
  else if (count > 0)
    count = __builtin_amdgcn_readfirstlane(beam_first<true>(list, count, a.n_out, floor, keys[wid]));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const uint64_t mine = lane < count ? keys[wid][lane] : 0ull;
  if (lane == 0) redn[wid] = count;
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    #pragma unroll
    for (int w = 0; w < W; ++w) n += redn[w];
    a.parts[slot] = BeamPart{m, s, (uint32_t)min(n, a.n_out), 0u};
  }
  // the waves' lists, ranked by counting
  int rank = 0;
  #pragma unroll 1
  for (int w = 0; w < W; ++w) {
    const int n = redn[w];
    #pragma unroll 4
    for (int i = 0; i < n; ++i) rank += keys[w][i] > mine;
  }
  if (lane < count && rank < a.n_out) a.cand[slot * a.n_out + rank] = mine;
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
  __shared__ float lse[kBeamMax], base[kBeamMax];  // base: the beams' scores
  __shared__ uint32_t state[kBeamMax];  // 0: no candidates, 1: its parts' candidates, 2: finished
  __shared__ uint32_t red[W];
  __shared__ uint32_t counter;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int row0 = b * a.K;
  const float ninf = -__builtin_inff();
  if (tid == 0) counter = 0u;
  // A list: what a part kept of a beam, in order (a finished beam has one
  // candidate, the first of its first list).  Q threads take a list, thread
  // `sub` every Q-th place from its own, and the lists beyond 512 / Q in further
  // rounds.  Lists go round the waves, so that beams and places are spread
  // evenly over them.  The first kFinishHeld a thread are loaded ahead of the
  // beams' sums (places that hold no candidate too: dropped by their count).
  // First a bound from the threads' first candidates, then all that reach it:
  // the work follows n_out and the lists, not their product (32 f32 rows of
  // 151,936 as one request's beams, 64 candidates: the whole step 28 us, with
  // every place of every list rated 107).
  const int lists = a.K * a.n_parts;
  const int qs = a.list_threads, Q = 1 << qs, turn = lane * W + wid;
  auto sub_of = [&](int list) { return (turn + list + (list >> 3)) & (Q - 1); };
  auto cand = [&](int list, int place) { return a.cand[((int64_t)row0 * a.n_parts + list) * a.n_out + place]; };
  auto kept = [&](int list) { return (int)a.parts[(int64_t)row0 * a.n_parts + list].n; };
  const int list0 = turn >> qs, sub0 = sub_of(list0);
  uint64_t held[kFinishHeld];
  int kept0 = 0;
  if (list0 < lists) kept0 = kept(list0);
  #pragma unroll
  for (int j = 0; j < kFinishHeld; ++j)
    held[j] = list0 < lists && sub0 + j * Q < a.n_out ? cand(list0, sub0 + j * Q) : 0ull;
  for (int k = wid; k < a.K; k += W) {
    const int row = row0 + k;
    const BeamFlag flag(a, row);
    const float c = flag.score;
    const BeamPart* pp = a.parts + (int64_t)row * a.n_parts;
    float m = ninf, s = 0.f;
    for (int i = lane; i < a.n_parts; i += 64) {
      const BeamPart p = pp[i];
      // (a first pair needs no scaling: m is -inf)
      const float hi = fmaxf(m, p.m);
      s = beam_finite(hi) ? s * __expf(m - hi) + p.sum * __expf(p.m - hi) : 0.f;
      m = hi;
    }
    const float top = beam_wave_max(m);
    uint32_t st = 0u;
    float l = 0.f;
    if (beam_finite(c)) {
      if (flag.finished()) {
        st = 2u;
      } else if (beam_finite(top)) {
        l = top + logf(beam_wave_sum(s * __expf(m - top)));
        st = 1u;
      }
    }
    if (lane == 0) { lse[k] = l; base[k] = c; state[k] = st; }
  }
  __syncthreads();
  auto rated = [&](int list, int place, uint64_t lo, int n) -> BeamCand {
    const int k = list / a.n_parts;
    const uint32_t st = state[k];
    BeamCand x{0ull, 0ull};
    if (st == 0u) return x;
    float score = base[k];
    if (st == 2u) {
      if (place != 0 || list != k * a.n_parts) return x;
      lo = 0xffffffffu - a.eos;
    } else {
      if (place >= n) return x;
      score += beam_okey_inv((uint32_t)(lo >> 32)) - lse[k];
      if (!beam_finite(score)) return x;
    }
    x.lo = lo;
    x.hi = ((uint64_t)beam_okey(score) << 32) | (0xffffffffu - (uint32_t)k);
    return x;
  };
  auto score_of = [](const BeamCand& x) { return (uint32_t)(x.hi >> 32); };
  // a bound that n_out of the threads' first candidates reach
  uint32_t best[1] = {0u};
  BeamCand mine[kFinishHeld];
  #pragma unroll
  for (int j = 0; j < kFinishHeld; ++j) {
    mine[j] = BeamCand{0ull, 0ull};
    if (list0 < lists && sub0 + j * Q < a.n_out) mine[j] = rated(list0, sub0 + j * Q, held[j], kept0);
  }
  best[0] = score_of(mine[0]);
  for (int list = list0 + (kFinishThreads >> qs); list < lists; list += kFinishThreads >> qs)
    best[0] = max(best[0], score_of(rated(list, sub_of(list), cand(list, sub_of(list)), kept(list))));
  uint32_t bound = max(beam_bound<1, W>(best, a.n_out, 0u, red), 1u);
  auto offer = [&](const BeamCand& x) {
    if (score_of(x) < bound) return false;
    const uint32_t o = atomicAdd(&counter, 1u);
    if (o < (uint32_t)kFinishSlots) slots[o] = x;
    return true;
  };
  for (;;) {
    // all that reach it: a list's scores descend
    bool more = true;
    #pragma unroll
    for (int j = 0; j < kFinishHeld; ++j)
      if (more) more = offer(mine[j]);
    int place = more ? sub0 + kFinishHeld * Q : a.n_out;
    for (int list = list0; list < lists;) {
      if (place < a.n_out && offer(rated(list, place, cand(list, place), kept(list)))) {
        place += Q;
      } else {
        list += kFinishThreads >> qs;
        place = sub_of(list);
      }
    }
    __syncthreads();
    if (counter <= (uint32_t)kFinishSlots) break;
    // too many: again, with a bound that n_out of those that were kept reach
    const uint32_t key[1] = {score_of(slots[tid])};
    const uint32_t higher = beam_bound<1, W>(key, a.n_out, 0u, red);
    if (higher <= bound) break;
    bound = higher;
    __syncthreads();
    if (tid == 0) counter = 0u;
    __syncthreads();
  }
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
    // ranks by counting, eight lanes a candidate
    for (int j = tid >> 3; j < n; j += kFinishThreads / 8) {
      const BeamCand x = slots[j];
      int rank = 0;
      #pragma unroll 4
      for (int i = tid & 7; i < n; i += 8) rank += beam_before(slots[i], x) ? 1 : 0;
      rank = beam_sum8(rank);
      if ((tid & 7) == 0 && rank < a.n_out) put(rank, x);
    }
    return;
  }
  // many equal scores: one candidate after another
  const int total = lists * a.n_out;
  BeamCand prev{~0ull, ~0ull};
  for (int r = 0; r < keep; ++r) {
    BeamCand top{0ull, 0ull};
    for (int i = tid; i < total; i += kFinishThreads) {
      const int list = i / a.n_out, place = i - list * a.n_out;
      const BeamCand x = rated(list, place, cand(list, place), kept(list));
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

// How a row is cut: into parts of kTileElems while all rows' parts are few, or
// into parts of `tiles` streamed tiles (a multiple of four: one a wave) that
// leave about four workgroups a CU.  Whole steps of 8 candidates, us, cut to
// parts and streamed:
//   4 rows of 151,936 (152 parts): f32 11.2 and 12.6, bf16 11.3 and 15.5
//   384 rows of 50,257 (4,992): 23.2 and 26.2, 23.0 and 27.3
//   512 rows of 50,257 (6,656): 28.3 and 28.7, 27.1 and 27.1
//   1,024 rows of 32,000 (8,192): 36.0 and 28.7, 35.2 and 27.5
// A mask costs the streaming kernel more (its words come with every tile):
//   1,024 rows of 50,257 (13,312): 60.2 and 58.5, 54.3 and 59.0
//   512 rows of 151,936 (19,456): 82.6 and 74.2, 69.7 and 76.1
//   768 rows of 128,256 (24,576): 101.1 and 104.1, 88.8 and 76.9
constexpr int kBeamFewParts = 6144, kBeamFewMasked = 3 * kBeamFewParts;
struct BeamCut {
  int tiles;  // 0: parts of kTileElems
  int parts;
};
BeamCut beam_cut(int64_t rows, int V, int dtype, bool masked) {
  const int64_t len = (int64_t)V + 7;  // (up to 7 elements before the row's start)
  const int64_t few = (len + kTileElems - 1) / kTileElems;
  if (rows * few <= (masked ? kBeamFewMasked : kBeamFewParts)) return BeamCut{0, (int)few};
  const int64_t tile = 64 * (dtype == HI_ROCM_DTYPE_F32 ? 16 : 32), steps = (len + 4 * tile - 1) / (4 * tile);
  const int64_t want = std::max<int64_t>(1, std::min(steps, (1024 + rows - 1) / rows));
  const int64_t tiles = 4 * ((steps + want - 1) / want);
  return BeamCut{(int)tiles, (int)((len + tiles * tile - 1) / (tiles * tile))};
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
void launch_parts(const BeamArgs& a, int rows, hipStream_t st) {
  const dim3 grid((unsigned)a.n_parts, (unsigned)rows), threads(kPartThreads);
  if (a.tiles == 0) hipLaunchKernelGGL(beam_tile_kernel<DT>, grid, threads, 0, st, a);
  else if (a.mask) hipLaunchKernelGGL((beam_part_kernel<DT, true>), grid, threads, 0, st, a);
  else hipLaunchKernelGGL((beam_part_kernel<DT, false>), grid, threads, 0, st, a);
}

// ---- states ---------------------------------------------------------------

typedef uint32_t reorder_u32x4 __attribute__((ext_vector_type(4)));

struct ReorderArgs {
  const char* src;
  char* dst;
  const int32_t* parents;  // [batch][K]
  const int32_t* lengths;  // [batch] or null
  int K;
  int64_t outer, mid, positions, pos_bytes;
  int64_t outer_stride, row_stride, mid_stride;
  int64_t blocks;  // workgroups of a piece
};

// One thread owns U units (16, 4, 2 or 1 bytes) of all K rows of a request: it
// reads what the rows need before it writes any of them, so dst may be src.
// A workgroup stays in one piece (outer and mid index) of one request, so that
// nothing but the column is divided per thread.  Bound by the bytes read and
// written: 1.3 GB of 8 requests' 8 beams 270 us, 4.9 TB/s, what a copy reaches.
template <typename T, int KM, int U>
__global__ void __launch_bounds__(256) beam_reorder_kernel(ReorderArgs a) {
  const int b = blockIdx.y;
  int64_t len = a.positions;
  if (a.lengths) {
    const int64_t l = a.lengths[b];
    len = l < 0 ? 0 : (l < len ? l : len);
  }
  const int64_t units = (len * a.pos_bytes + (int64_t)sizeof(T) - 1) / (int64_t)sizeof(T);
  const int64_t piece = blockIdx.x / (uint32_t)a.blocks, col0 = (int64_t)(blockIdx.x % (uint32_t)a.blocks) * (256 * U);
  if (col0 >= units) return;
  const int64_t o = piece / a.mid, m = piece - o * a.mid;
  const int64_t at = o * a.outer_stride + m * a.mid_stride + (int64_t)b * a.K * a.row_stride;
  const T* src = reinterpret_cast<const T*>(a.src + at) + col0 + threadIdx.x;
  T* dst = reinterpret_cast<T*>(a.dst + at) + col0 + threadIdx.x;
  const int64_t row = a.row_stride / (int64_t)sizeof(T);
  const bool same = a.src == a.dst;
  bool in[U];
  #pragma unroll
  for (int u = 0; u < U; ++u) in[u] = col0 + u * 256 + (int)threadIdx.x < units;
  T v[KM][U];
  bool moves[KM];
  #pragma unroll
  for (int j = 0; j < KM; ++j) {
    moves[j] = false;
    if (j < a.K) {
      const int p = a.parents[b * a.K + j];
      const int q = p < 0 || p >= a.K ? j : p;  // (a parent outside the request: the row stays)
      moves[j] = !same || q != j;
      if (moves[j]) {
        #pragma unroll
        for (int u = 0; u < U; ++u)
          if (in[u]) v[j][u] = src[q * row + u * 256];
      }
    }
  }
  #pragma unroll
  for (int j = 0; j < KM; ++j)
    if (moves[j]) {
      #pragma unroll
      for (int u = 0; u < U; ++u)
        if (in[u]) dst[j * row + u * 256] = v[j][u];
    }
}

template <typename T, int KM, int U>
void launch_reorder_rows(ReorderArgs a, int batch, hipStream_t st) {
  const int64_t units = (a.positions * a.pos_bytes + (int64_t)sizeof(T) - 1) / (int64_t)sizeof(T);
  a.blocks = (units + 256 * U - 1) / (256 * U);
  const dim3 grid((unsigned)(a.outer * a.mid * a.blocks), (unsigned)batch);
  hipLaunchKernelGGL((beam_reorder_kernel<T, KM, U>), grid, dim3(256), 0, st, a);
}

// Up to 16 units a thread.  us with the fitting kernel and the next larger one:
// K = 4 (537 MB) 143 and 146, K = 8 (1,074 MB) 331 and 356, K = 16 (2,147 MB)
// 776 and 837.
template <typename T>
void launch_reorder(const ReorderArgs& a, int batch, hipStream_t st) {
  if (a.K <= 4) launch_reorder_rows<T, 4, 4>(a, batch, st);
  else if (a.K <= 8) launch_reorder_rows<T, 8, 2>(a, batch, st);
  else if (a.K <= 16) launch_reorder_rows<T, 16, 1>(a, batch, st);
  else launch_reorder_rows<T, 32, 1>(a, batch, st);
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
                    "hi_rocm_beam_workspace_bytes: more than 32 beams, 64 outputs, 65535 rows or 2^23 tokens");
  int64_t slots = 0;
  for (int b = 1; b <= max_batch; ++b)
    for (int dtype : {HI_ROCM_DTYPE_F32, HI_ROCM_DTYPE_BF16})
      for (bool masked : {false, true})
        slots = std::max(slots, (int64_t)b * beams * beam_cut((int64_t)b * beams, vocab, dtype, masked).parts);
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
  if (beams > kBeamMax || n_out > kBeamMaxOut || vocab > kMaxVocab || (int64_t)batch * beams > kBeamMaxRows)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_beam_select: more than 32 beams, 64 outputs, 65535 rows or 2^23 tokens");
  const int rows = batch * beams;
  BeamArgs a;
  memset(&a, 0, sizeof(a));
  const BeamCut cut = beam_cut(rows, vocab, dtype, mask_words != nullptr);
  a.tiles = cut.tiles;
  a.n_parts = cut.parts;
  while ((2 << a.list_threads) * beams * a.n_parts <= kFinishThreads && (1 << a.list_threads) < n_out) ++a.list_threads;
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
  if (dtype == HI_ROCM_DTYPE_F32) launch_parts<HI_ROCM_DTYPE_F32>(a, rows, (hipStream_t)stream);
  else launch_parts<HI_ROCM_DTYPE_BF16>(a, rows, (hipStream_t)stream);
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
  if (beams > kBeamMax || batch > kBeamMaxRows)
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
  // the widest unit in which all rows start and end: 537 MB in 4 rows a request
  // 126 us; from an address on 4 bytes 136, on 2 bytes 169 (by bytes three times
  // the first)
  const int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  // (a launch holds less than 2^32 threads; outer * mid * blocks: each below 2^46)
  const int64_t blocks = ((piece + unit - 1) / unit + 255) / 256, most = UINT32_MAX / 256;
  if (outer > most || mid > most / outer || blocks > most / (outer * mid))
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_beam_reorder: more than 2^24 pieces of 256 units a row");
  if (unit == 16) launch_reorder<reorder_u32x4>(a, batch, (hipStream_t)stream);
  else if (unit == 4) launch_reorder<uint32_t>(a, batch, (hipStream_t)stream);
  else if (unit == 2) launch_reorder<uint16_t>(a, batch, (hipStream_t)stream);
  else launch_reorder<uint8_t>(a, batch, (hipStream_t)stream);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "beam reorder launch");
}

}  // extern "C"
