// Speculative-decoding verification of sampled drafts (the rejection rule of
// speculative sampling, docs/deepseek-v4-spec-decode-plan.md:95-102 names it; the
// reference implements only the greedy acceptance, spec_verify.hip here).
//
// Request b has drafts t_0 .. t_{k-1}, the target's probabilities p_0 .. p_k after
// each and the draft model's q_0 .. q_{k-1} (without them a draft was certain: q_i
// is 1 at t_i).  With the given random numbers u:
//     draft i is accepted  <=>  u_i q_i(t_i) < p_i(t_i)
//     n = the first draft not accepted, or k
//     r = max(p_n - q_n, 0), or p_k after k accepted drafts
//     token = the least j with r_0 + .. + r_j > u_last (r_0 + .. + r_{V-1})
// Emitted tokens then follow p exactly.  The product of two f32 is exact in f64,
// and all sums are f64: no rounding that a test could see decides a token.
//
// One launch: every workgroup finds n (a gather of two values a draft), sums r
// over its part of the one row of p and q that counts, and the request's last
// workgroup finds the token's part among the sums and the token in that part.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "hi_rocm.h"
#include "sampler_internal.h"
#include "wave_ops.h"

namespace hi_rocm {
namespace {

constexpr int kSampledWaves = 4;
constexpr int kSampledThreads = 64 * kSampledWaves;
constexpr size_t kSampledLine = 128;
// Values a lane has in flight of a row: enough to stream, few enough that their
// f64 sums do not take longer than the loads' latency.  us with 4, 8 .. 64 KB parts
// of f32 (8, 16, 32, 64 values a lane): 1 request of 151,936 6.2, 6.0, 6.7, 8.5; 64
// requests 17.4, 15.4, 16.4, 17.9; bf16 (16, 32, 64, 128 values) 6.5, 6.9, 8.8, 12.5
// and 13.6, 13.1, 14.6, 19.2.
constexpr int kSampledValues = 16;
constexpr int kSampledSpan = kSampledThreads * kSampledValues;  // values of a part

struct SampledArgs {
  const void* target;
  int64_t target_batch, target_row;  // values
  const void* draft;                 // or null
  int64_t draft_batch, draft_row;
  const uint32_t* tokens;    // [batch][K]
  const int32_t* lengths;    // [batch] or null
  const float* uniforms;     // [batch][K + 1]
  uint32_t* out_tokens;      // [batch][K + 1]
  int32_t* out_count;        // [batch]
  uint32_t* counters;        // [batch], a line each, 0 between calls
  double* sums;              // [batch][parts * kSampledWaves]
  int V, K, parts;
};

__device__ __forceinline__ float sampled_value(const float* p) { return *p; }
__device__ __forceinline__ float sampled_value(const __bf16* p) { return (float)*p; }

// n values of a row from p on, 16 bytes a lane and load, range-checked.  Rows of
// bf16 may start in the middle of a word: their loads begin a half earlier and
// are shifted.
template <typename T>
struct SampledRow {
  static constexpr int E = 16 / sizeof(T);
  __amdgpu_buffer_rsrc_t rs;
  bool odd;
  __device__ __forceinline__ void open(const T* p, int n) {
    odd = sizeof(T) == 2 && ((uintptr_t)p & 2) != 0;
    const uint32_t bytes = n > 0 ? (uint32_t)n * sizeof(T) + (odd ? 2u : 0u) : 0u;
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)((uintptr_t)p & ~(uintptr_t)3), 0, (int)((bytes + 3u) & ~3u), kBufferConfig);
  }
  __device__ __forceinline__ i32x4_t load(int at) const {
    const int byte = at * (int)sizeof(T);
    i32x4_t v = __builtin_amdgcn_raw_buffer_load_b128(rs, byte, 0, 0);
    if (sizeof(T) == 2 && odd) {
      const uint32_t next = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, byte + 16, 0, 0);
      const uint32_t w[5] = {(uint32_t)v[0], (uint32_t)v[1], (uint32_t)v[2], (uint32_t)v[3], next};
      #pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = (int)(w[j] >> 16 | w[j + 1] << 16);
    }
    return v;
  }
  static __device__ __forceinline__ float get(const i32x4_t& v, int e) {
    if constexpr (sizeof(T) == 4) return __int_as_float(v[e]);
    else return __uint_as_float(e & 1 ? (uint32_t)v[e >> 1] & 0xffff0000u : (uint32_t)v[e >> 1] << 16);
  }
};

// What is drawn from: the row of p, the row of q to take off (null: none), and
// the certain draft (or none, V).
template <typename T>
struct SampledRest {
  const T* p;
  const T* q;
  uint32_t certain;
};
__device__ __forceinline__ double sampled_rest(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 ? d : 0.0;  // (NaN: nothing)
}
template <typename T>
__device__ __forceinline__ double sampled_at(const SampledRest<T>& s, int j) {
  const float q = s.q != nullptr ? sampled_value(s.q + j) : (uint32_t)j == s.certain ? 1.f : 0.f;
  return sampled_rest(sampled_value(s.p + j), q);
}

// Sums over the wave's lanes up to each, by moves within the registers (six
// steps through LDS took 0.2 us more a sum).
template <int CTRL, int ROW_MASK = 0xf, bool BC = false>
__device__ __forceinline__ double sampled_up(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = dpp32<CTRL, ROW_MASK, BC>(0u, (uint32_t)b), hi = dpp32<CTRL, ROW_MASK, BC>(0u, (uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double sampled_wave_scan(double v) {
  v += sampled_up<kDppShr1, 0xf, true>(v);
  v += sampled_up<kDppShr1 + 1, 0xf, true>(v);
  v += sampled_up<kDppShr1 + 3, 0xf, true>(v);
  v += sampled_up<kDppShr1 + 7, 0xf, true>(v);
  v += sampled_up<kDppBcast15, 0xa>(v);
  v += sampled_up<kDppBcast31, 0xc>(v);
  return v;
}
constexpr int kSampledHeld = 2;

// A wave's sum, as its workgroup wrote it (from wherever it ran).
__device__ __forceinline__ double sampled_sum(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct SampledLds {
  double wave[kSampledWaves];
  int first[kSampledWaves], positive[kSampledWaves];
  double base;
  int at, last;
};

// Among the threads' shares v of the workgroup's sum, in thread order from base
// on, the first that passes `bound` (without one the last above 0, or -1), and
// in `before` the sum before it.  All threads get both.
__device__ __forceinline__ int sampled_pick(SampledLds& L, double v, double base, double bound, double& before) {
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  double incl = sampled_wave_scan(v);
  __syncthreads();
  if (lane == 63) L.wave[wid] = incl;
  __syncthreads();
  double start = base;
  for (int w = 0; w < wid; ++w) start += L.wave[w];
  incl += start;
  const uint64_t over = __ballot(v > 0.0 && incl > bound), some = __ballot(v > 0.0);
  if (lane == 0) {
    L.first[wid] = over != 0ull ? wid * 64 + __builtin_ctzll(over) : -1;
    L.positive[wid] = some != 0ull ? wid * 64 + 63 - __builtin_clzll(some) : -1;
  }
  __syncthreads();
  int at = -1;
  for (int w = kSampledWaves - 1; w >= 0; --w) at = L.first[w] >= 0 ? L.first[w] : at;
  for (int w = kSampledWaves - 1; at < 0 && w >= 0; --w) at = L.positive[w];
  if (tid == at) L.base = incl - v;
  __syncthreads();
  before = L.base;
  __syncthreads();
  return at;
}

// The token among [j0, j1), at most kSampledThreads * per values.
template <typename T>
__device__ __forceinline__ int sampled_token(SampledLds& L, const SampledRest<T>& s, int j0, int j1, double base,
                                             double bound) {
  const int per = (j1 - j0 + kSampledThreads - 1) / kSampledThreads;
  const int a = min(j0 + (int)threadIdx.x * per, j1), b = min(a + per, j1);
  double sum = 0.0;
  for (int j = a; j < b; ++j) sum += sampled_at(s, j);
  double before;
  const int at = sampled_pick(L, sum, base, bound, before);
  if (at < 0) return -1;
  if ((int)threadIdx.x == at) {
    int token = -1;
    for (int j = a; j < b; ++j) {
      const double r = sampled_at(s, j);
      if (!(r > 0.0)) continue;
      token = j;
      before += r;
      if (before > bound) break;
    }
    L.at = token;
  }
  __syncthreads();
  return L.at;
}

// The token from p alone, by one workgroup: where nothing is left of p - q
// (which a rejection rules out but for roundings of p and q).
template <typename T>
__device__ __forceinline__ int sampled_alone(SampledLds& L, const SampledRest<T>& s, int V, float u) {
  constexpr int kTile = kSampledThreads * 8;
  double total = 0.0;
  for (int j = threadIdx.x; j < V; j += kSampledThreads) total += sampled_at(s, j);
  total = sampled_wave_scan(total);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) L.wave[threadIdx.x >> 6] = total;
  __syncthreads();
  total = 0.0;
  for (int w = 0; w < kSampledWaves; ++w) total += L.wave[w];
  const double bound = (double)u * total;
  double base = 0.0;
  int token = -1;
  for (int j0 = 0; j0 < V; j0 += kTile) {
    const int j1 = min(j0 + kTile, V);
    double sum = 0.0;
    for (int j = j0 + (int)threadIdx.x; j < j1; j += kSampledThreads) sum += sampled_at(s, j);
    sum = sampled_wave_scan(sum);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) L.wave[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kSampledWaves; ++w) sum += L.wave[w];
    if (sum > 0.0) {
      const int t = sampled_token(L, s, j0, j1, base, bound);
      token = t >= 0 ? t : token;
      if (base + sum > bound) break;
    }
    base += sum;
    __syncthreads();
  }
  return token;
}

template <typename T>
__global__ void __launch_bounds__(kSampledThreads) spec_sampled_kernel(SampledArgs a) {
  __shared__ SampledLds L;
  constexpr int E = SampledRow<T>::E, I = kSampledValues / E, kWave = 64 * kSampledValues;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / (uint32_t)a.parts, part = blockIdx.x % (uint32_t)a.parts;
  const int V = a.V, K = a.K;
  const T* target = (const T*)a.target + (int64_t)b * a.target_batch;
  const T* draft = a.draft != nullptr ? (const T*)a.draft + (int64_t)b * a.draft_batch : nullptr;
  // The accepted drafts, by every wave for itself (no load waits for the number
  // of drafts: those past it are looked at in vain).
  int k = K;
  if (a.lengths != nullptr) k = min(max(a.lengths[b], 0), K);
  const float u = a.uniforms[(int64_t)b * (K + 1) + K];
  int n = K;
  uint32_t certain = (uint32_t)V;
  for (int i0 = 0; i0 < K; i0 += 64) {
    const int i = i0 + lane;
    bool rejected = false;
    uint32_t t = (uint32_t)V;
    if (i < K) {
      t = a.tokens[(int64_t)b * K + i];
      const float ui = a.uniforms[(int64_t)b * (K + 1) + i];
      rejected = true;
      if (t < (uint32_t)V) {
        const float p = sampled_value(target + i * a.target_row + t);
        const float q = draft != nullptr ? sampled_value(draft + i * a.draft_row + t) : 1.f;
        rejected = !((double)ui * (double)q < (double)p);
      }
    }
    const uint64_t no = __ballot(rejected);
    if (no != 0ull) {
      const int l = __builtin_ctzll(no);
      n = i0 + l;
      certain = (uint32_t)__builtin_amdgcn_readlane((int)t, l);
      break;
    }
  }
  n = __builtin_amdgcn_readfirstlane(min(n, k));
  SampledRest<T> s;
  s.p = target + n * a.target_row;
  s.q = n < k && draft != nullptr ? draft + n * a.draft_row : nullptr;
  s.certain = n < k && draft == nullptr ? certain : (uint32_t)V;
  // this wave's part
  const int j0 = min((part * kSampledWaves + wid) * kWave, V), j1 = min(j0 + kWave, V);
  SampledRow<T> rp, rq;
  rp.open(s.p + j0, j1 - j0);
  rq.open(s.q != nullptr ? s.q + j0 : s.p + j0, s.q != nullptr ? j1 - j0 : 0);
  i32x4_t pv[I], qv[I];
  #pragma unroll
  for (int i = 0; i < I; ++i) {
    pv[i] = rp.load((i * 64 + lane) * E);
    qv[i] = rq.load((i * 64 + lane) * E);  // (none: out of range, zero)
  }
  double sum = 0.0;
  #pragma unroll
  for (int i = 0; i < I; ++i) {
    #pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = j0 + (i * 64 + lane) * E + e;
      const float q = (uint32_t)j == s.certain ? 1.f : SampledRow<T>::get(qv[i], e);
      const double r = sampled_rest(SampledRow<T>::get(pv[i], e), q);
      sum += j < j1 ? r : 0.0;
    }
  }
  sum = sampled_wave_scan(sum);
  double* sums = a.sums + (int64_t)b * a.parts * kSampledWaves;
  if (lane == 63)
    __hip_atomic_store(sums + part * kSampledWaves + wid, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // The request's last workgroup goes on.  All that it reads of the others are
  // the sums, written and read past the caches that one XCD has to itself (atomics
  // of the agent's scope), and each wave's has arrived (vmcnt 0) before its
  // workgroup counts: no fence, whose write-back of an XCD's L2 costs more than
  // the whole call.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) {
    uint32_t* counter = a.counters + b * (kSampledLine / 4);
    L.last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
             (uint32_t)(a.parts - 1);
    if (L.last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!L.last) return;
  // Each thread's waves, up to kSampledHeld of them in registers.
  const int pieces = a.parts * kSampledWaves, per = (pieces + kSampledThreads - 1) / kSampledThreads;
  const int c0 = min(tid * per, pieces), c1 = min(c0 + per, pieces);
  double held[kSampledHeld], mine = 0.0;
  #pragma unroll
  for (int i = 0; i < kSampledHeld; ++i) held[i] = c0 + i < c1 ? sampled_sum(sums + c0 + i) : 0.0;
  #pragma unroll
  for (int i = 0; i < kSampledHeld; ++i) mine += held[i];
  for (int c = c0 + kSampledHeld; c < c1; ++c) mine += sampled_sum(sums + c);
  double total = sampled_wave_scan(mine);
  if (lane == 63) L.wave[wid] = total;
  __syncthreads();
  total = 0.0;
  #pragma unroll
  for (int w = 0; w < kSampledWaves; ++w) total += L.wave[w];
  int token = -1;
  if (total > 0.0) {
    const double bound = (double)u * total;
    double before;
    const int at = sampled_pick(L, mine, 0.0, bound, before);
    // (at is a thread: some share is above 0)
    if (tid == at) {
      int found = c0;
      bool over = false;
      auto look = [&](int c, double v) {
        if (over || !(v > 0.0)) return;
        found = c;
        L.base = before;
        over = before + v > bound;
        before += v;
      };
      #pragma unroll
      for (int i = 0; i < kSampledHeld; ++i) look(c0 + i, held[i]);
      for (int c = c0 + kSampledHeld; c < c1 && !over; ++c) look(c, sampled_sum(sums + c));
      L.at = found;
    }
    __syncthreads();
    const int c = __builtin_amdgcn_readfirstlane(L.at);
    const double base = L.base;
    // that wave's values again, a load a thread
    static_assert(kSampledThreads * E >= kWave, "one load covers a wave's part");
    const int w0 = min(c * kWave, V), w1 = min(w0 + kWave, V);
    rp.open(s.p + w0, w1 - w0);
    rq.open(s.q != nullptr ? s.q + w0 : s.p + w0, s.q != nullptr ? w1 - w0 : 0);
    const i32x4_t p4 = rp.load(tid * E), q4 = rq.load(tid * E);  // (behind the part: out of range, zero)
    double r[E], share = 0.0;
    #pragma unroll
    for (int e = 0; e < E; ++e) {
      const int j = w0 + tid * E + e;
      const float q = (uint32_t)j == s.certain ? 1.f : SampledRow<T>::get(q4, e);
      const double v = sampled_rest(SampledRow<T>::get(p4, e), q);
      r[e] = j < w1 ? v : 0.0;
      share += r[e];
    }
    const int in = sampled_pick(L, share, base, bound, before);
    if (tid == in) {
      bool over = false;
      #pragma unroll
      for (int e = 0; e < E; ++e) {
        if (over || !(r[e] > 0.0)) continue;
        token = w0 + tid * E + e;
        before += r[e];
        over = before > bound;
      }
      L.at = token;
    }
    __syncthreads();
    token = L.at;
  } else {
    s.q = nullptr;
    s.certain = (uint32_t)V;
    token = sampled_alone(L, s, V, u);
  }
  token = max(token, 0);
  for (int i = tid; i <= K; i += kSampledThreads) {
    uint32_t t = HI_ROCM_SPEC_NO_TOKEN;
    if (i < n) t = a.tokens[(int64_t)b * K + i];
    else if (i == n) t = (uint32_t)token;
    a.out_tokens[(int64_t)b * (K + 1) + i] = t;
  }
  if (tid == 0) a.out_count[b] = n + 1;
}

int sampled_parts(int vocab) { return (int)(((int64_t)vocab + kSampledSpan - 1) / kSampledSpan); }

// The first half of a workspace holds the counters, which are 0 between calls, a
// cache line each: counts on one line take some 5 ns after each other, wherever
// they come from (64 requests of 151,936 f32: 15 us, with counters side by side 27).
// The second holds the sums.  So the counters' place depends on the workspace's
// size alone, not on a call's batch and vocabulary.
constexpr int kSampledMaxBatch = 65535;
size_t sampled_half(int64_t batch, int vocab) {
  const size_t sums = (size_t)batch * sampled_parts(vocab) * kSampledWaves * 8;
  return (std::max((size_t)batch * kSampledLine, sums) + kSampledLine - 1) / kSampledLine * kSampledLine;
}

template <typename T>
hipError_t launch_sampled(SampledArgs& a, int batch, hipStream_t st) {
  a.parts = sampled_parts(a.V);
  const int64_t groups = (int64_t)batch * a.parts;
  if (groups > UINT32_MAX / kSampledThreads) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((spec_sampled_kernel<T>), dim3((unsigned)groups), dim3(kSampledThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace
}  // namespace hi_rocm

using namespace hi_rocm;

extern "C" {

int hi_rocm_spec_sampled_workspace_bytes(int max_batch, int vocab, size_t* out_bytes) {
  if (max_batch <= 0 || vocab <= 0 || out_bytes == nullptr)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_spec_sampled_workspace_bytes: invalid arguments");
  if (max_batch > kSampledMaxBatch || vocab > kMaxVocab)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_spec_sampled_workspace_bytes: more than 65535 requests or 2^23 tokens");
  *out_bytes = 2 * sampled_half(max_batch, vocab);
  return HI_ROCM_OK;
}

int hi_rocm_spec_verify_sampled(const void* target_probs, int dtype, int batch, int max_draft, int vocab,
                                int64_t target_batch_stride, int64_t target_row_stride, const void* draft_probs,
                                int64_t draft_batch_stride, int64_t draft_row_stride, const uint32_t* draft_tokens,
                                const int32_t* draft_len, const float* uniforms, uint32_t* out_tokens,
                                int32_t* out_count, void* workspace, size_t workspace_bytes, void* stream) {
  if (target_probs == nullptr || batch <= 0 || max_draft < 0 || vocab <= 0 ||
      (max_draft > 0 && draft_tokens == nullptr) || uniforms == nullptr || out_tokens == nullptr ||
      out_count == nullptr || workspace == nullptr || (dtype != HI_ROCM_DTYPE_F32 && dtype != HI_ROCM_DTYPE_BF16) ||
      target_batch_stride < 0 || target_row_stride < 0 ||
      (draft_probs != nullptr && (draft_batch_stride < 0 || draft_row_stride < 0)))
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_spec_verify_sampled: invalid arguments");
  const int size = dtype == HI_ROCM_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)target_probs % size != 0 || (uintptr_t)draft_probs % size != 0)
    return api_fail(HI_ROCM_ERR_ARGS, "hi_rocm_spec_verify_sampled: probabilities not aligned to their type");
  if (batch > kSampledMaxBatch || vocab > kMaxVocab || max_draft > 65535)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED,
                    "hi_rocm_spec_verify_sampled: more than 65535 requests or drafts, or 2^23 tokens");
  if ((uintptr_t)workspace % 16 != 0 || workspace_bytes < 2 * sampled_half(batch, vocab))
    return api_fail(HI_ROCM_ERR_ARGS,
                    "hi_rocm_spec_verify_sampled: workspace not on 16 bytes, or too small "
                    "(hi_rocm_spec_sampled_workspace_bytes)");
  SampledArgs a;
  a.target = target_probs;
  a.target_batch = target_batch_stride;
  a.target_row = target_row_stride;
  a.draft = max_draft > 0 ? draft_probs : nullptr;
  a.draft_batch = draft_batch_stride;
  a.draft_row = draft_row_stride;
  a.tokens = draft_tokens;
  a.lengths = draft_len;
  a.uniforms = uniforms;
  a.out_tokens = out_tokens;
  a.out_count = out_count;
  a.counters = (uint32_t*)workspace;
  a.sums = (double*)((char*)workspace + workspace_bytes / (2 * kSampledLine) * kSampledLine);
  a.V = vocab;
  a.K = max_draft;
  const hipError_t e = dtype == HI_ROCM_DTYPE_F32 ? launch_sampled<float>(a, batch, (hipStream_t)stream)
                                                  : launch_sampled<__bf16>(a, batch, (hipStream_t)stream);
  if (e == hipErrorInvalidConfiguration)
    return api_fail(HI_ROCM_ERR_UNSUPPORTED, "hi_rocm_spec_verify_sampled: too many requests and tokens for one launch");
  return e == hipSuccess ? HI_ROCM_OK : api_hip_fail(e, "spec sampled launch");
}

}  // extern "C"
