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
// A workgroup takes LG_SLICE tokens of one row: it counts the row's history
// into LDS (one counter per token of the slice), then streams the slice.  The
// counters are integers, so the order of the LDS atomics does not show: plain
// counts in 32 bits, decayed ones in 64-bit steps of 2^-40 (every occurrence
// adds at least one step, so `seen` is a count above zero; a history of 2^23
// tokens cannot overflow).
#include <type_traits>

#include "sample_common.h"

namespace rwkv7mi {

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_SLICE = 4096;
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

}  // namespace

template <typename TI, typename TO, bool DECAY>
__global__ __launch_bounds__(LG_THREADS) void logits_kernel(const LgArgs A) {
  using C = std::conditional_t<DECAY, unsigned long long, uint32_t>;
  __shared__ C count[LG_SLICE];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  const int c0 = (int)blockIdx.x * LG_SLICE, len = min(LG_SLICE, A.V - c0);
  const bool hist = A.history != nullptr;
  float theta = 1.f, pres = 0.f, freq = 0.f;
  if (hist) {
    theta = lg_get(A.repetition, row);
    pres = lg_get(A.presence, row);
    freq = lg_get(A.frequency, row);
    for (int i = tid; i < LG_SLICE; i += LG_THREADS) count[i] = 0;
    __syncthreads();
    const int64_t n = A.lengths ? min((int64_t)max(A.lengths[row], 0), A.L) : A.L;
    const double d = DECAY ? fmin(fmax((double)lg_get(A.decay, row), 0.0), 1.0) : 1.0;
    for (int64_t i = tid; i < n; i += LG_THREADS) {
      const int64_t t = lg_token(A, row, i) - c0;  // (tokens outside the vocabulary count nowhere)
      if (t < 0 || t >= len) continue;
      if constexpr (DECAY) {
        const double w = rint(pow(d, (double)(n - 1 - i)) * 0x1p40);
        atomicAdd(&count[t], (unsigned long long)fmax(w, 1.0));
      } else {
        atomicAdd(&count[t], 1u);
      }
    }
    __syncthreads();
  }
  const TI* x = static_cast<const TI*>(A.x) + row * A.ldx + c0;
  TO* out = static_cast<TO*>(A.out) + row * A.ldo + c0;
  const float* bias = A.bias ? A.bias + row * A.ldb + c0 : nullptr;
  const uint32_t* allowed = A.allowed ? A.allowed + row * A.lda + c0 / 32 : nullptr;
  float bv = -__builtin_inff();
  int bi = INT32_MAX;
  for (int i = tid; i < len; i += LG_THREADS) {
    float v = to_f32(x[i]);
    if (hist) {
      const C c = count[i];
      if (c) {
        const float occ = DECAY ? (float)((double)c * 0x1p-40) : (float)c;
        v = v > 0.f ? v / theta : v * theta;
        v -= pres + freq * occ;
      }
    }
    if (bias) v += bias[i];
    if (allowed && !((allowed[i >> 5] >> (i & 31)) & 1u)) v = -__builtin_inff();
    const TO r = from_f32<TO>(v);
    out[i] = r;
    const float f = to_f32(r);
    if (am_better(f, c0 + i, bv, bi)) bv = f, bi = c0 + i;
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

extern "C" size_t rwkv7mi_process_logits_workspace_bytes(int64_t rows, int64_t V) {
  if (rows <= 0 || V <= 0) return 0;
  return (size_t)(rows * ((V + LG_SLICE - 1) / LG_SLICE)) * 8u;
}

extern "C" int rwkv7mi_process_logits(const void* x, int64_t rows, int64_t V, int64_t ldx, int dtype, void* out,
                                      int64_t ldo, int out_dtype, void* history, int history_bits, int64_t ldh,
                                      int64_t L, int* lengths, const float* const* penalties, const float* penalty,
                                      int decayed, const float* bias, int64_t ldb, const uint32_t* allowed, int64_t lda,
                                      int64_t* next, int64_t* next2, int append, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const std::string w("process_logits");
  if (rows < 0 || V <= 0 || ldx < 0 || (rows > 1 && ldo < V)) return fail(RWKV7MI_EINVAL, w + ": bad shape");
  if (!valid_dtype(dtype) || !(out_dtype == dtype || out_dtype == RWKV7MI_F32))
    return fail(RWKV7MI_EINVAL, w + ": the output has the logits' type or fp32");
  if (rows > 65535 || V > INT32_MAX - LG_SLICE) return fail(RWKV7MI_EINVAL, w + ": too large");
  if (history_bits != 32 && history_bits != 64) return fail(RWKV7MI_EINVAL, w + ": 32- or 64-bit history entries");
  if (history && (L < 0 || ldh < 0 || L > LG_MAX_HISTORY))
    return fail(RWKV7MI_EINVAL, w + ": bad history (at most 2^23 tokens a row)");
  if (history && (!penalties || !penalty)) return fail(RWKV7MI_EINVAL, w + ": null penalties");
  if (ldb < 0 || lda < 0) return fail(RWKV7MI_EINVAL, w + ": bad stride");
  if (rows == 0) return RWKV7MI_OK;
  if (!x || !out) return fail(RWKV7MI_EINVAL, w + ": null pointer");
  if (next2 && !next) return fail(RWKV7MI_EINVAL, w + ": the second copy of the tokens needs the first");
  if (append && (!history || !lengths || !next || (rows > 1 && ldh < L)))
    return fail(RWKV7MI_EINVAL, w + ": appending needs a history of separate rows, its lengths and the tokens");
  const int nb = (int)((V + LG_SLICE - 1) / LG_SLICE);
  if (next && (!workspace || workspace_bytes < (size_t)(rows * nb) * 8u || (reinterpret_cast<uintptr_t>(workspace) & 7)))
    return fail(RWKV7MI_ESIZE, w + ": workspace missing, unaligned or smaller than "
                                   "rwkv7mi_process_logits_workspace_bytes");
  LgArgs a{x, out, ldx, ldo, (int)V, history_bits == 64};
  // (penalties that change nothing need no counts)
  const bool idle = history && !penalties[0] && !penalties[1] && !penalties[2] && penalty[0] == 1.f &&
                    penalty[1] == 0.f && penalty[2] == 0.f;
  if (history && L > 0 && !idle) {
    a.history = history;
    a.lengths = lengths;
    a.ldh = ldh;
    a.L = L;
    LgScalar* s[4] = {&a.repetition, &a.presence, &a.frequency, &a.decay};
    for (int i = 0; i < 4; ++i) *s[i] = LgScalar{penalties[i], penalty[i]};
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
