// The logits step of a served row: penalties for repeated tokens, a bias, a
// grammar mask, and the greedy token.
//
// For token t of a row with history h[0 .. n-1] (h[n-1] the newest):
//   c = sum over i with h[i] = t of decay^(n - 1 - i)
//   seen (some h[i] = t):  l = l > 0 ? l / repetition : l * repetition
//                          l = l - (presence + frequency c)
//   l = l + bias[t];  not allowed: l = -inf
// in fp32, rounded once to the output type.
//
// A workgroup takes 8 tokens a lane of one row: it counts the row's history into LDS (one
// counter per token of the slice), then streams the slice, one 16-byte run of logits a
// lane (two of fp32).  Runs are cut at 16-byte boundaries of the row's memory, so
// rows of any length and offset load whole; what they write and add is vectorised
// where it lies alike.  The counters are integers, so the order of the LDS atomics does
// not show: plain counts in 32 bits, decayed ones in 64-bit steps of 2^-40 (every
// occurrence adds at least one step, so `seen` is a count above zero; a history of 2^23
// tokens cannot overflow).
//
// Latency- and issue-bound: the history's loads, then one run; every workgroup of a row
// reads its whole history, from L2, and a wave has a decayed entry of its slice in most
// of its loads, each with fp64 work.  64 rows of 65536 fp16 logits, mask and bias (19
// MB), with the token: 25.7 us behind 4000-token histories and decay, 17.1 without
// decay, 13.0 behind 100 tokens without mask and bias; one row of 500 tokens 7.9.  (1024
// lanes and 8192 tokens a workgroup: 2 us less for 64 x 65536, 7 more for 64 x 50277,
// 17.4 here.  The decayed entries gathered in LDS and weighed by all lanes at once:
// 32.5.)
#include <type_traits>

#include "sample_common.h"

namespace rwkv7mi {

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_SLICE = 2048;
constexpr int LG_FLIGHT = 4;  // history entries a lane loads at once (8: registers for 7 waves only)
constexpr int64_t LG_MAX_HISTORY = 1 << 23;

// one value a row: values[row], or the same for every row
struct LgScalar {
  const float* values;
  float value;
};
__device__ __forceinline__ float lg_get(const LgScalar& s, int64_t row) { return s.values ? s.values[row] : s.value; }

struct LgArgs {
  const void* x;
  void* out;
  int64_t ldx, ldo;
  int V, bits64;  // bits64: 64-bit history entries
  const void* history;
  const int* lengths;
  int64_t ldh, L;
  LgScalar repetition, presence, frequency, decay;
  const float* bias;
  int64_t ldb;
  const uint32_t* allowed;
  int64_t lda;
  float* pv;  // the slices' best values and indices (null: no token wanted)
  int* pi;
};

__device__ __forceinline__ int64_t lg_token(const LgArgs& A, int64_t row, int64_t i) {
  const int64_t at = row * A.ldh + i;
  return A.bits64 ? static_cast<const int64_t*>(A.history)[at] : (int64_t) static_cast<const int*>(A.history)[at];
}

// elements by which a row starts behind a 16-byte boundary
template <typename T>
__device__ __forceinline__ int lg_shift(const T* p) { return (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T)); }

}  // namespace

template <typename TI, typename TO, bool DECAY>
__global__ __launch_bounds__(LG_THREADS) void logits_kernel(const LgArgs A) {
  using C = std::conditional_t<DECAY, unsigned long long, uint32_t>;
  constexpr int E = 16 / (int)sizeof(TI), RUNS = LG_SLICE / LG_THREADS / E;  // elements of a run, runs of a lane
  __shared__ __align__(16) C count[LG_SLICE];
  __shared__ double log_decay;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  const TI* x = static_cast<const TI*>(A.x) + row * A.ldx;
  const int shift = lg_shift(x);
  const int c0 = (int)blockIdx.x * LG_SLICE - shift;  // the slice's first token (before the row in the first slice)
  // this lane's logits
  float v[RUNS][E];
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int i = c0 + E * (LG_THREADS * u + tid);
    if (i >= 0 && i + E <= A.V) {
      uint4 d = *reinterpret_cast<const uint4*>(x + i);
      const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (sizeof(TI) == 4)
          v[u][e] = __uint_as_float(w[e]);
        else
          v[u][e] = to_f32(__builtin_bit_cast(TI, (uint16_t)(w[e / 2] >> (16 * (e & 1)))));
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[u][e] = i + e >= 0 && i + e < A.V ? to_f32(x[i + e]) : 0.f;
    }
  }
  const bool hist = A.history != nullptr;
  float theta = 1.f, pres = 0.f, freq = 0.f;
  if (hist) {
    theta = lg_get(A.repetition, row);
    pres = lg_get(A.presence, row);
    freq = lg_get(A.frequency, row);
#pragma unroll
    for (int i = 0; i < LG_SLICE / LG_THREADS; ++i) count[LG_THREADS * i + tid] = 0;
    if (DECAY && tid < 64)  // (one wave: fp64 instructions are slow; its lanes write the same)
      log_decay = log2(fmin(fmax((double)lg_get(A.decay, row), 0.0), 1.0));
    __syncthreads();
    const int64_t n = A.lengths ? min((int64_t)max(A.lengths[row], 0), A.L) : A.L;
    const double ld = DECAY ? log_decay : 0.0;
    // tokens of the slice that are in the vocabulary: width of them from c0 + lo
    const int lo = max(-c0, 0), width = max(min(LG_SLICE, A.V - c0) - lo, 0);
    for (int64_t i0 = tid; i0 < n; i0 += LG_FLIGHT * LG_THREADS) {
      int64_t t[LG_FLIGHT];
#pragma unroll
      for (int k = 0; k < LG_FLIGHT; ++k) {
        const int64_t i = i0 + LG_THREADS * k;
        t[k] = i < n ? lg_token(A, row, i) : -1;
      }
      int at[LG_FLIGHT];  // (in 32 bits before the fp64 work: registers for 8 waves)
#pragma unroll
      for (int k = 0; k < LG_FLIGHT; ++k) {
        const uint64_t d = (uint64_t)t[k] - (uint64_t)(c0 + lo);
        at[k] = d < (uint64_t)width ? lo + (int)d : -1;
      }
#pragma unroll
      for (int k = 0; k < LG_FLIGHT; ++k) {
        const int o = at[k];
        if (o < 0) continue;
        if constexpr (DECAY) {
          const int age = (int)(n - 1 - i0) - LG_THREADS * k;
          // (past 2^-41 one step; decay 0 counts the newest alone)
          const double w = age ? exp2(fmax((double)age * ld, -100.0) + 40.0) : 0x1p40;
          atomicAdd(&count[o], (unsigned long long)fmax(rint(w), 1.0));
        } else {
          atomicAdd(&count[o], 1u);
        }
      }
    }
    __syncthreads();
  }
  TO* out = static_cast<TO*>(A.out) + row * A.ldo;
  const float* bias = A.bias ? A.bias + row * A.ldb : nullptr;
  const uint32_t* allowed = A.allowed ? A.allowed + row * A.lda : nullptr;
  const bool vout = ((reinterpret_cast<uintptr_t>(out) - shift * sizeof(TO)) & 15) == 0;
  const bool vbias = ((reinterpret_cast<uintptr_t>(bias) - shift * sizeof(float)) & 15) == 0;
  float bv = -__builtin_inff();
  int bi = INT32_MAX;
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int o = E * (LG_THREADS * u + tid), i = c0 + o;
    if (i + E <= 0 || i >= A.V) continue;
    const bool whole = i >= 0 && i + E <= A.V;
    if (hist) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const C c = count[o + e];
        if (c) {
          const float occ = DECAY ? (float)((double)c * 0x1p-40) : (float)c;
          float l = v[u][e];
          l = l > 0.f ? l / theta : l * theta;
          v[u][e] = l - (pres + freq * occ);
        }
      }
    }
    if (bias) {
      if (whole && vbias) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
          const float4 q = *reinterpret_cast<const float4*>(bias + i + e);
          v[u][e] += q.x, v[u][e + 1] += q.y, v[u][e + 2] += q.z, v[u][e + 3] += q.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (i + e >= 0 && i + e < A.V) v[u][e] += bias[i + e];
      }
    }
    if (allowed) {
      // the run's bits from the one or two words that hold them
      const int first = max(i, 0), w0 = first >> 5, w1 = (min(i + E, A.V) - 1) >> 5;
      const uint64_t two = allowed[w0] | (uint64_t)allowed[w1] << 32;
      const uint32_t bits = (uint32_t)(two >> (first & 31)) << (first - i);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(bits >> e & 1u)) v[u][e] = -__builtin_inff();
    }
    TO r[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      r[e] = from_f32<TO>(v[u][e]);
      const float f = to_f32(r[e]);
      if (i + e >= 0 && i + e < A.V && am_better(f, i + e, bv, bi)) bv = f, bi = i + e;
    }
    if (whole && vout) {
      constexpr int Q = E * (int)sizeof(TO) / 16;
      uint32_t d[4 * Q];
#pragma unroll
      for (int q = 0; q < 4 * Q; ++q) {
        if constexpr (sizeof(TO) == 4)
          d[q] = __float_as_uint(r[q]);
        else
          d[q] = (uint32_t)__builtin_bit_cast(uint16_t, r[2 * q]) | (uint32_t)__builtin_bit_cast(uint16_t, r[2 * q + 1]) << 16;
      }
#pragma unroll
      for (int q = 0; q < Q; ++q)
        reinterpret_cast<uint4*>(out + i)[q] = make_uint4(d[4 * q], d[4 * q + 1], d[4 * q + 2], d[4 * q + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e >= 0 && i + e < A.V) out[i + e] = r[e];
    }
  }
  if (!A.pv) return;
  am_wave_best(bv, bi);
  __shared__ float sv[LG_THREADS / 64];
  __shared__ int si[LG_THREADS / 64];
  if ((tid & 63) == 0) {
    sv[tid >> 6] = bv;
    si[tid >> 6] = bi;
  }
  __syncthreads();
  if (tid == 0) {
    float v = sv[0];
    int i = si[0];
#pragma unroll
    for (int w = 1; w < LG_THREADS / 64; ++w)
      if (am_better(sv[w], si[w], v, i)) v = sv[w], i = si[w];
    A.pv[row * gridDim.x + blockIdx.x] = v;
    A.pi[row * gridDim.x + blockIdx.x] = i;
  }
}

// One wave a row: the best of its slices, and (append) the token behind the
// row's history where there is room.
__global__ __launch_bounds__(64) void logits_token_kernel(const float* __restrict__ pv, const int* __restrict__ pi,
                                                          int nb, int64_t* next, int64_t* next2, void* history,
                                                          int* lengths, int64_t ldh, int64_t L, int bits64) {
  const int64_t row = blockIdx.x;
  float bv = -__builtin_inff();
  int bi = INT32_MAX;
  for (int j = threadIdx.x; j < nb; j += 64) {
    const float v = pv[row * nb + j];
    const int i = pi[row * nb + j];
    if (am_better(v, i, bv, bi)) bv = v, bi = i;
  }
  am_wave_best(bv, bi);
  if (threadIdx.x) return;
  next[row] = bi;
  if (next2) next2[row] = bi;
  if (!history) return;
  const int n = max(lengths[row], 0);
  if (n >= L) return;
  if (bits64)
    static_cast<int64_t*>(history)[row * ldh + n] = bi;
  else
    static_cast<int*>(history)[row * ldh + n] = bi;
  lengths[row] = n + 1;
}

}  // namespace rwkv7mi

using namespace rwkv7mi;

// slices of a row, which starts up to 7 elements behind a boundary
static int64_t lg_slices(int64_t V) { return (V + 7 + LG_SLICE - 1) / LG_SLICE; }

extern "C" size_t rwkv7mi_process_logits_workspace_bytes(int64_t rows, int64_t V) {
  if (rows <= 0 || V <= 0) return 0;
  return (size_t)(rows * lg_slices(V)) * 8u;
}

extern "C" int rwkv7mi_process_logits(const void* x, int64_t rows, int64_t V, int64_t ldx, int dtype, void* out,
                                      int64_t ldo, int out_dtype, void* history, int history_bits, int64_t ldh,
                                      int64_t L, int* lengths, const float* repetition_rows, float repetition,
                                      const float* presence_rows, float presence, const float* frequency_rows,
                                      float frequency, const float* decay_rows, float decay, const float* bias, int64_t ldb, const uint32_t* allowed, int64_t lda,
                                      int64_t* next, int64_t* next2, int append, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const std::string w("process_logits");
  if (rows < 0 || V <= 0 || ldx < 0 || (rows > 1 && ldo < V)) return fail(RWKV7MI_EINVAL, w + ": bad shape");
  if (!valid_dtype(dtype) || !(out_dtype == dtype || out_dtype == RWKV7MI_F32))
    return fail(RWKV7MI_EINVAL, w + ": the output has the logits' type or fp32");
  if (rows > 65535 || V > INT32_MAX - 65536) return fail(RWKV7MI_EINVAL, w + ": too large");
  if (history_bits != 32 && history_bits != 64) return fail(RWKV7MI_EINVAL, w + ": 32- or 64-bit history entries");
  if (history && (L < 0 || ldh < 0 || L > LG_MAX_HISTORY))
    return fail(RWKV7MI_EINVAL, w + ": bad history (at most 2^23 tokens a row)");
  if (ldb < 0 || lda < 0) return fail(RWKV7MI_EINVAL, w + ": bad stride");
  if (rows == 0) return RWKV7MI_OK;
  if (!x || !out) return fail(RWKV7MI_EINVAL, w + ": null pointer");
  if (next2 && !next) return fail(RWKV7MI_EINVAL, w + ": the second copy of the tokens needs the first");
  if (append && (!history || !lengths || !next || (rows > 1 && ldh < L)))
    return fail(RWKV7MI_EINVAL, w + ": appending needs a history of separate rows, its lengths and the tokens");
  // (rows that all start on a boundary need no slice more)
  const int64_t es = dtype == RWKV7MI_F32 ? 4 : 2;
  const bool straight = !(reinterpret_cast<uintptr_t>(x) & 15) && (rows == 1 || (ldx * es) % 16 == 0);
  const int nb = (int)lg_slices(straight ? V - 7 : V);
  if (next && (!workspace || workspace_bytes < (size_t)(rows * nb) * 8u || (reinterpret_cast<uintptr_t>(workspace) & 7)))
    return fail(RWKV7MI_ESIZE, w + ": workspace missing, unaligned or smaller than "
                                   "rwkv7mi_process_logits_workspace_bytes");
  LgArgs a{x, out, ldx, ldo, (int)V, history_bits == 64};
  // (penalties that change nothing need no counts)
  const bool idle = !repetition_rows && !presence_rows && !frequency_rows && repetition == 1.f && presence == 0.f &&
                    frequency == 0.f;
  const bool decayed = decay_rows || decay != 1.f;
  if (history && L > 0 && !idle) {
    a.history = history;
    a.lengths = lengths;
    a.ldh = ldh;
    a.L = L;
    a.repetition = LgScalar{repetition_rows, repetition};
    a.presence = LgScalar{presence_rows, presence};
    a.frequency = LgScalar{frequency_rows, frequency};
    a.decay = LgScalar{decay_rows, decay};
  }
  a.bias = bias;
  a.ldb = ldb;
  a.allowed = allowed;
  a.lda = lda;
  a.pv = next ? static_cast<float*>(workspace) : nullptr;
  a.pi = next ? reinterpret_cast<int*>(a.pv + rows * nb) : nullptr;
  const dim3 grid((unsigned)nb, (unsigned)rows);
  const int rc = dispatch_dtype(dtype, [&](auto ti) {
    using TI = decltype(ti);
    const auto go = [&](auto to) {
      using TO = decltype(to);
      if (decayed)
        hipLaunchKernelGGL((logits_kernel<TI, TO, true>), grid, dim3(LG_THREADS), 0, as_stream(stream), a);
      else
        hipLaunchKernelGGL((logits_kernel<TI, TO, false>), grid, dim3(LG_THREADS), 0, as_stream(stream), a);
      return check_launch("logits_kernel");
    };
    return out_dtype == dtype ? go(ti) : go(float{});
  });
  if (rc || !next) return rc;
  hipLaunchKernelGGL(logits_token_kernel, dim3((unsigned)rows), dim3(64), 0, as_stream(stream), a.pv, a.pi, nb, next,
                     next2, append ? history : nullptr, lengths, ldh, L, a.bits64);
  return check_launch("logits_token_kernel");
}
