// Beam search's step on the device: the best candidates of a prompt over its
// beams and the vocabulary, and what follows from them.
//
// For prompt b, beam k with running score s and logits x[0 .. V-1]:
//   value(k, t) = s + (x[t] - lse),  lse = m + log sum_t exp(x[t] - m)
// in 64 bits (so that which of two close candidates comes first does not hang on
// fp32's last bits), rounded once to fp32.  The M best of the K V values, best
// first, equal ones by (k, t).  A row that holds NaN or +inf, or whose score is
// one, is NaN throughout, and NaN ranks first, as in the argmax; a token of
// logit -inf, and every token of a row that is -inf throughout or whose score
// is, has the value -inf.
//
// beam_slice_kernel: one workgroup per slice of a row, one pass over the logits
// (runs of 16 bytes, cut at 16-byte boundaries of the row's memory, held in
// registers): the slice's maximum and sum of exponentials, and its M best
// logits (a row's score and lse do not change the order inside it).  The lanes'
// maxima give a bound: at least M values of the slice reach the M-th largest of
// them, found bit by bit with ballots; the few that do are gathered in LDS and
// ranked by counting.  -inf is never gathered: a masked row costs no more than
// another.  Values in numbers that LDS does not hold (long ties, sorted rows)
// are drawn one by one instead.
//
// beam_merge_kernel: one workgroup per prompt joins the slices' sums to lse, in
// 64 bits, and selects among their K S M candidates the same way; the step's
// bookkeeping (ends, hypotheses, places of the beams, token rows) follows in the
// same workgroup.
#include "common.h"

namespace rwkv7mi {

namespace {

constexpr int BM_THREADS = 256;
constexpr int BM_CAP = 1024;      // candidates that a workgroup gathers
constexpr int BM_MOST = 128;      // candidates of a prompt
constexpr int BM_ENDS = 8;        // end tokens

struct BmState {
  int64_t* tokens;
  int* lengths;
  float* scores;
  int* prompt_lengths;
  int64_t* finished_tokens;
  int* finished_lengths;
  float* finished_scores;
  uint8_t* done;
};

struct BmArgs {
  const void* x;
  int64_t ldx;
  int V, beams, S, M, normalized;
  const float* scores;
  // the slices' results: [rows][S][M] values (high) and beams and tokens (low), best first;
  // [rows][S] maxima and sums
  uint64_t* got;
  float2* sums;
  float* out_scores;  // the selection's own outputs (null in a step)
  int64_t *out_tokens, *out_rows;
};

struct BmStep {
  BmState in, out;
  int64_t room, pad;
  int64_t *next, *rows;
  double penalty;
  int early, ends, in_place;
  int64_t end[BM_ENDS];
};

// a float's order as an unsigned number (-0 as 0)
__device__ __forceinline__ uint32_t bm_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float bm_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ uint64_t bm_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);
  return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double bm_value(uint64_t k) {
  return __longlong_as_double((long long)(k >> 63 ? k ^ 0x8000000000000000ull : ~k));
}
constexpr uint32_t BM_NONE = 0x007fffffu;  // the key of -inf: nothing to choose
// a slice's candidate: the logit's key, the beam (7 bits), the token (23)
__device__ __forceinline__ uint64_t bm_pack(uint32_t key, int beam, int token) {
  return (uint64_t)key << 32 | (uint32_t)(beam << 23 | token);
}
// what decides between equal values: the beam (7 bits), the logit, the token (23)
__device__ __forceinline__ uint64_t bm_place(uint64_t c) {
  return (c & 0x3f800000u) << 32 | (uint64_t) ~(uint32_t)(c >> 32) << 23 | (c & 0x7fffffu);
}
__device__ __forceinline__ int bm_beam(uint64_t p) { return (int)(p >> 55); }
__device__ __forceinline__ int bm_token(uint64_t p) { return (int)(p & 0x7fffff); }

__device__ __forceinline__ uint32_t bm_wave_max(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

// The largest t such that M of the n keys in LDS (64 Q of them, all above
// BM_NONE or equal to it) reach t, as far as bits LOW and up tell; BM_NONE + 1 where
// fewer than M are above BM_NONE.  One wave.
template <int Q, int LOW>
__device__ __forceinline__ uint32_t bm_bound(const uint32_t* keys, int M) {
  uint32_t k[Q];
#pragma unroll
  for (int q = 0; q < Q; ++q) k[q] = keys[64 * q + (threadIdx.x & 63)];
  uint32_t t = 0;
  for (int b = 31; b >= LOW; --b) {
    const uint32_t c = t | 1u << b;
    int n = 0;
#pragma unroll
    for (int q = 0; q < Q; ++q) n += __popcll(__ballot(k[q] >= c));
    if (n >= M) t = c;
    if (n == M) break;
  }
  return max(t, BM_NONE + 1);
}

}  // namespace

// RUNS 16-byte runs a lane.
template <typename T, int RUNS>
__global__ __launch_bounds__(BM_THREADS) void beam_slice_kernel(const BmArgs A) {
  constexpr int E = 16 / (int)sizeof(T), SLICE = BM_THREADS * RUNS * E;
  constexpr int LOW = std::is_same<T, __half>::value ? 13 : sizeof(T) == 2 ? 16 : 0;  // bits that T's values have
  __shared__ uint64_t got[BM_CAP];
  __shared__ uint32_t top[BM_THREADS];
  __shared__ uint32_t bound, wave_top[BM_THREADS / 64];
  __shared__ float wave_sum_[BM_THREADS / 64];
  __shared__ int count;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(A.x) + row * A.ldx;
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int c0 = (int)blockIdx.x * SLICE - shift;  // the slice's first token (before the row in the first slice)
  float v[RUNS][E];
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int i = c0 + E * (BM_THREADS * u + tid);
    if (i >= 0 && i + E <= A.V) {
      const uint4 d = *reinterpret_cast<const uint4*>(x + i);
      const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (sizeof(T) == 4)
          v[u][e] = __uint_as_float(w[e]);
        else
          v[u][e] = to_f32(__builtin_bit_cast(T, (uint16_t)(w[e / 2] >> (16 * (e & 1)))));
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[u][e] = i + e >= 0 && i + e < A.V ? to_f32(x[i + e]) : -__builtin_inff();
    }
  }
  if (tid == 0) count = 0;
  float run_best[RUNS], best = -__builtin_inff();
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    run_best[u] = v[u][0];
#pragma unroll
    for (int e = 1; e < E; ++e) run_best[u] = fmaxf(run_best[u], v[u][e]);
    best = fmaxf(best, run_best[u]);
  }
  const uint32_t mine = bm_key(best);
  top[tid] = mine;
  const uint32_t wtop = bm_wave_max(mine);
  if ((tid & 63) == 0) wave_top[tid >> 6] = wtop;
  __syncthreads();
  uint32_t all = wave_top[0];
#pragma unroll
  for (int w = 1; w < BM_THREADS / 64; ++w) all = max(all, wave_top[w]);
  if (tid < 64) {
    const uint32_t t = bm_bound<BM_THREADS / 64, LOW>(top, A.M);
    if (tid == 0) bound = t;
  }
  const float m = bm_value(all);
  // NaN and +inf make the sum NaN (a slice of -inf and NaN alone: asked for)
  float s = 0.f;
  if (all > BM_NONE) {
#pragma unroll
    for (int u = 0; u < RUNS; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f((v[u][e] - m) * 1.44269504f);
  } else {
#pragma unroll
    for (int u = 0; u < RUNS; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) s = v[u][e] != v[u][e] ? __builtin_nanf("") : s;
  }
  s = wave_sum(s);
  if ((tid & 63) == 0) wave_sum_[tid >> 6] = s;
  __syncthreads();
  const uint32_t at_least = bound;
  const float reach = bm_value(at_least);
  const int64_t slice = row * A.S + blockIdx.x;
  const int beam = (int)(row % A.beams);
  if (tid == 0) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < BM_THREADS / 64; ++w) sum += wave_sum_[w];
    A.sums[slice] = make_float2(m, sum);
  }
  uint64_t* out = A.got + slice * A.M;
  const int t0 = c0 + E * tid;
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    if (!(run_best[u] >= reach)) continue;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (v[u][e] >= reach) {
        const int p = atomicAdd(&count, 1);
        if (p < BM_CAP) got[p] = (uint64_t)bm_key(v[u][e]) << 32 | (uint32_t) ~(t0 + E * BM_THREADS * u + e);
      }
  }
  __syncthreads();
  const int n = count;
  if (n <= BM_CAP) {
    for (int i = tid; i < n; i += BM_THREADS) {
      const uint64_t k = got[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += got[j] > k;
      if (r < A.M) out[r] = bm_pack((uint32_t)(k >> 32), beam, (int)~(uint32_t)k);
    }
    for (int r = n + tid; r < A.M; r += BM_THREADS) out[r] = 0;
    return;
  }
  // too many reach the bound: M times the best below the last
  uint64_t last = ~0ull;
  for (int r = 0; r < A.M; ++r) {
    uint64_t k = 0;
#pragma unroll
    for (int u = 0; u < RUNS; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint64_t c = (uint64_t)bm_key(v[u][e]) << 32 | (uint32_t) ~(t0 + E * BM_THREADS * u + e);
        if (v[u][e] >= reach && c < last && c > k) k = c;
      }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t c = __shfl_xor((unsigned long long)k, o, 64);
      k = max(k, c);
    }
    __syncthreads();
    if ((tid & 63) == 0) got[tid >> 6] = k;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < BM_THREADS / 64; ++w) k = max(k, got[w]);
    last = k;
    if (tid == 0) out[r] = bm_pack((uint32_t)(k >> 32), beam, (int)~(uint32_t)k);
  }
}

namespace {

struct BmBest {  // a prompt's candidates, best first
  float value[BM_MOST];
  int token[BM_MOST], beam[BM_MOST];
};

// the position of the q-th (from 0) clear bit of the first n of mask; n where there is none
__device__ __forceinline__ int bm_clear_bit(const uint64_t* mask, int n, int q) {
  for (int i = 0; i < n; ++i)
    if (!(mask[i >> 6] >> (i & 63) & 1) && q-- == 0) return i;
  return n;
}

// a row of n tokens by one wave, eight loads in flight
__device__ __forceinline__ void bm_copy(int64_t* dst, const int64_t* src, int n) {
  const int lane = threadIdx.x & 63;
  for (int i0 = lane; i0 < n; i0 += 512) {
    int64_t t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + 64 * u < n) t[u] = src[i0 + 64 * u];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (i0 + 64 * u < n) dst[i0 + 64 * u] = t[u];
  }
}

}  // namespace

__device__ void beam_bookkeeping(const BmArgs& A, const BmStep& P, const BmBest& best) {
  __shared__ int live[BM_MOST], place[BM_MOST], taken[BM_MOST];  // taken: the hypothesis of a slot, -1: as before
  __shared__ float hyp[BM_MOST], old[BM_MOST];
  __shared__ uint64_t used[2], kept[2];
  __shared__ int is_end[BM_MOST], twin[BM_MOST];
  const int tid = threadIdx.x, K = A.beams;
  const int64_t b = blockIdx.x, r0 = b * K;
  const bool was = P.in.done[b];
  const int len = P.in.lengths[r0], prompt = P.in.prompt_lengths[b];
  const bool full = len < 0 || len >= P.room;  // (no room: nothing can follow)
  const int waves = blockDim.x >> 6, wave = tid >> 6;
  const auto held = [&](int k) { return min(max(P.in.finished_lengths[r0 + k], 0), (int)P.room); };
  if (was || full) {
    if (!P.in_place)
      for (int j = wave; j < 2 * K; j += waves) {
        const int64_t at = (r0 + (j >> 1)) * P.room;
        if (j & 1)
          bm_copy(P.out.finished_tokens + at, P.in.finished_tokens + at, held(j >> 1));
        else
          bm_copy(P.out.tokens + at, P.in.tokens + at, min(max(len, 0), (int)P.room));
      }
    if (tid < K) {
      const int64_t r = r0 + tid;
      P.next[r] = P.pad;
      P.rows[r] = r;
      P.out.lengths[r] = P.in.lengths[r];
      P.out.scores[r] = P.in.scores[r];
      P.out.finished_lengths[r] = P.in.finished_lengths[r];
      P.out.finished_scores[r] = P.in.finished_scores[r];
    }
    if (tid == 0) {
      P.out.done[b] = 1;
      P.out.prompt_lengths[b] = prompt;
    }
    return;
  }
  const double span = pow((double)max(len + 1 - prompt, 1), P.penalty);
  if (tid < K) old[tid] = P.in.finished_scores[r0 + tid], taken[tid] = -1;
  if (tid < 2) used[tid] = kept[tid] = 0;
  const bool last = len + 1 >= P.room;  // the rows are full behind this token: all texts end
  if (tid < A.M) {
    bool end = false;
    for (int e = 0; e < P.ends; ++e) end |= best.token[tid] == P.end[e];
    is_end[tid] = end && best.value[tid] > -__builtin_inff();
    if (tid < K) hyp[tid] = (end || last) && best.value[tid] > -__builtin_inff() ? (float)((double)best.value[tid] / span)
                                                                                 : -__builtin_inff();
  }
  __syncthreads();
  if (tid < A.M && !is_end[tid]) {  // the first K that do not end live on
    int r = 0;
    for (int j = 0; j < tid; ++j) r += !is_end[j];
    if (r < K) live[r] = tid;
  }
  if (tid < K) {
    // the K best of the hypotheses so far and those that end here, earlier ones first
    const float o = old[tid], h = hyp[tid];
    int ro = 0, rh = 0;
    for (int j = 0; j < K; ++j) {
      ro += (old[j] > o || (old[j] == o && j < tid)) + (hyp[j] > o);
      rh += (old[j] >= h) + (hyp[j] > h || (hyp[j] == h && j < tid));
    }
    if (ro < K) atomicOr((unsigned long long*)&kept[tid >> 6], 1ull << (tid & 63));
    place[tid] = h > -__builtin_inff() && rh < K;  // (as a flag; places of the beams below)
  }
  __syncthreads();
  if (tid < K && place[tid]) {
    int q = 0;
    for (int j = 0; j < tid; ++j) q += place[j];
    const int slot = bm_clear_bit(kept, K, q);
    if (slot < K) taken[slot] = tid;
  }
  if (tid < K) atomicOr((unsigned long long*)&used[best.beam[live[tid]] >> 6], 1ull << (best.beam[live[tid]] & 63));
  __syncthreads();
  if (tid < K) {
    int t = 0;
    for (int j = 0; j < tid; ++j) t |= best.beam[live[j]] == best.beam[live[tid]];
    twin[tid] = t;
  }
  __syncthreads();
  if (tid < K) {
    // a beam's first child keeps its row, the others take the rows that are left
    int q = 0;
    for (int j = 0; j < tid; ++j) q += twin[j];
    place[tid] = twin[tid] ? bm_clear_bit(used, K, q) : best.beam[live[tid]];
  }
  __syncthreads();
  // the texts: a wave a row; hypotheses first: in place, a row whose only child ended may be taken
  for (int k = wave; k < K; k += waves) {
    const int h = taken[k];
    int64_t* dst = P.out.finished_tokens + (r0 + k) * P.room;
    if (h >= 0)
      bm_copy(dst, P.in.tokens + (r0 + best.beam[h]) * P.room, len);
    else if (!P.in_place)
      bm_copy(dst, P.in.finished_tokens + (r0 + k) * P.room, held(k));
  }
  if (P.in_place) __syncthreads();
  for (int i = wave; i < K; i += waves) {
    const int c = live[i], k = place[i];
    if (!P.in_place || k != best.beam[c])
      bm_copy(P.out.tokens + (r0 + k) * P.room, P.in.tokens + (r0 + best.beam[c]) * P.room, len);
  }
  if (tid < K) {
    const int c = live[tid], h = taken[tid];
    const int64_t r = r0 + place[tid], f = r0 + tid;
    P.out.tokens[r * P.room + len] = best.token[c];
    P.next[r] = best.token[c];
    P.rows[r] = r0 + best.beam[c];
    P.out.lengths[r] = len + 1;
    P.out.scores[r] = best.value[c];
    if (h >= 0) {
      P.out.finished_tokens[f * P.room + len] = best.token[h];
      P.out.finished_lengths[f] = len + 1;
      P.out.finished_scores[f] = hyp[h];
    } else if (!P.in_place) {
      P.out.finished_lengths[f] = P.in.finished_lengths[f];
      P.out.finished_scores[f] = old[tid];
    }
  }
  if (tid < 64) {
    float worst = __builtin_inff();
    for (int k = tid; k < K; k += 64) worst = fminf(worst, taken[k] >= 0 ? hyp[taken[k]] : old[k]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) worst = fminf(worst, __shfl_xor(worst, o, 64));
    if (tid == 0) {
      // early 0: at the present length; 1: as soon as there are K hypotheses; 2: at the length that helps most
      const double ahead = P.early == 2 && P.penalty > 0 ? pow((double)max(P.room - prompt, (int64_t)1), P.penalty) : span;
      const bool over = P.early == 1 ? worst > -__builtin_inff()
                                     : !((float)((double)best.value[live[0]] / ahead) > worst);
      P.out.done[b] = over || last;
      P.out.prompt_lengths[b] = prompt;
    }
  }
}

template <int NT, bool STEP>
__global__ __launch_bounds__(NT) void beam_merge_kernel(const BmArgs A, const BmStep P) {
  constexpr int HOLD = 4;  // candidates that a lane keeps; further ones are read twice
  __shared__ uint64_t got[BM_CAP];
  __shared__ uint64_t got_at[BM_CAP];  // what decides where values are equal (bm_place), the least first
  __shared__ uint32_t top[256];
  __shared__ double lse[BM_MOST];
  __shared__ float score[BM_MOST];
  __shared__ int nan_rows[BM_MOST];  // the rows of NaN, in order; then the others
  __shared__ uint64_t poison[2];
  __shared__ uint32_t bound;
  __shared__ int count;
  __shared__ BmBest best;
  const int tid = threadIdx.x, lane = tid & 63, K = A.beams, M = A.M;
  const int64_t r0 = (int64_t)blockIdx.x * K;
  const int L = K * A.S, N = L * M;  // lists, candidates
  const uint64_t* list = A.got + r0 * A.S * M;
  // the candidates on their way while lse is formed
  uint64_t held[HOLD], head = 0;
#pragma unroll
  for (int i = 0; i < HOLD; ++i) held[i] = tid + NT * i < N ? list[tid + NT * i] : 0;
  if (tid < 256 && L <= 256 && tid / L < M) head = list[(tid % L) * M + tid / L];
  if (tid < 2) poison[tid] = 0;
  if (tid == 0) count = 0;
  __syncthreads();
  for (int k = tid >> 6; k < K; k += NT / 64) {  // a wave a row
    const float2* sums = A.sums + (r0 + k) * A.S;
    const float own = A.scores[r0 + k];
    float m = -__builtin_inff();
    for (int j = lane; j < A.S; j += 64) m = fmaxf(m, sums[j].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    double s = 0.0;
    for (int j = lane; j < A.S; j += 64) {
      const float2 q = sums[j];
      s += q.x > -__builtin_inff() ? (double)q.y * exp((double)q.x - (double)m) : (double)q.y;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) {
      if (s != s || !(own < __builtin_inff())) {
        atomicOr((unsigned long long*)&poison[k >> 6], 1ull << (k & 63));
        s = 1.0;
      }
      lse[k] = A.normalized || !(s > 0.0) ? 0.0 : (double)m + log(s);
      score[k] = own;
    }
  }
  __syncthreads();
  if (tid < K) {
    const bool p = poison[tid >> 6] >> (tid & 63) & 1;
    int q = 0, all = 0;
    for (int j = 0; j < K; ++j) {
      const bool o = poison[j >> 6] >> (j & 63) & 1;
      q += j < tid && o == p;
      all += o;
    }
    nan_rows[p ? q : all + q] = tid;
  }
  const int bad = __popcll(poison[0]) + __popcll(poison[1]);
  const int first = (int)min((int64_t)bad * A.V, (int64_t)M);  // NaN ranks first
  const int want = M - first;
  const auto value = [&](uint64_t c) {  // -inf: nothing to choose
    const int k = (int)(c >> 23 & 0x7f);
    if ((uint32_t)(c >> 32) <= BM_NONE || (poison[k >> 6] >> (k & 63) & 1)) return -__builtin_inf();
    return (double)score[k] + ((double)bm_value((uint32_t)(c >> 32)) - lse[k]);
  };
  // 256 candidates give the bound: the best of every list and, where lists are few, the next ones
  if (tid < 256) {
    uint32_t mine = bm_key((float)value(head));
    if (L > 256)
      for (int l = tid; l < L; l += 256) mine = max(mine, bm_key((float)value(list[(int64_t)l * M])));
    top[tid] = mine;
  }
  __syncthreads();
  if (tid < 64) {
    const uint32_t t = bm_bound<4, 0>(top, max(want, 1));
    if (tid == 0) bound = t;
  }
  __syncthreads();
  const uint32_t at_least = bound;
  const auto gather = [&](uint64_t c) {
    const double v = value(c);
    if (bm_key((float)v) >= at_least) {
      const int p = atomicAdd(&count, 1);
      if (p < BM_CAP) got[p] = bm_key(v), got_at[p] = bm_place(c);
    }
  };
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (held[i]) gather(held[i]);
  for (int j = tid + NT * HOLD; j < N; j += NT) gather(list[j]);
  __syncthreads();
  int n = count;
  const auto put = [&](int r, float v, int beam, int token) {
    best.value[r] = v;
    best.beam[r] = beam;
    best.token[r] = token;
  };
  if (n <= BM_CAP) {
    for (int i = tid; i < n; i += NT) {
      const uint64_t k = got[i], at = got_at[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += got[j] > k || (got[j] == k && got_at[j] < at);
      if (r < want) put(first + r, (float)bm_value(k), bm_beam(at), bm_token(at));
    }
  } else {
    uint64_t lk = ~0ull, la = 0;
    n = 0;
    for (int r = 0; r < want; ++r) {
      uint64_t k = 0, a = ~0ull;
      for (int j = tid; j < N; j += NT) {
        const double v = value(list[j]);
        if (!(v > -__builtin_inf())) continue;
        const uint64_t c = bm_key(v), at = bm_place(list[j]);
        if ((c < lk || (c == lk && at > la)) && (c > k || (c == k && at < a))) k = c, a = at;
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const uint64_t c = __shfl_xor((unsigned long long)k, o, 64), ca = __shfl_xor((unsigned long long)a, o, 64);
        if (c > k || (c == k && ca < a)) k = c, a = ca;
      }
      __syncthreads();
      if (lane == 0) got[tid >> 6] = k, got_at[tid >> 6] = a;
      __syncthreads();
      k = got[0], a = got_at[0];
#pragma unroll
      for (int w = 1; w < NT / 64; ++w)
        if (got[w] > k || (got[w] == k && got_at[w] < a)) k = got[w], a = got_at[w];
      if (k == 0) break;
      lk = k, la = a;
      ++n;
      if (tid == 0) put(first + r, (float)bm_value(k), bm_beam(a), bm_token(a));
    }
  }
  __syncthreads();
  // the NaN rows' tokens, and behind what can be chosen the -inf ones by their index
  if (tid < first) put(tid, __builtin_nanf(""), nan_rows[tid / A.V], tid % A.V);
  const int found = min(n, want);
  if (found < want && tid < 64) {
    int r = first + found;
    for (int j0 = 0; r < M; j0 += 64) {
      const int j = j0 + lane;
      const int ord = bad + j / A.V;  // (M values are there: bad V + others V >= M)
      const bool there = ord < K;
      const int beam = there ? nan_rows[ord] : 0, token = j % A.V;
      bool free = there;
      for (int i = 0; i < found && free; ++i) free = best.beam[first + i] != beam || best.token[first + i] != token;
      const uint64_t f = __ballot(free);
      const int p = r + __popcll(f & ((1ull << lane) - 1));
      if (free && p < M) put(p, -__builtin_inff(), beam, token);
      r += __popcll(f);
      if (!__any(there)) break;
    }
  }
  __syncthreads();
  if constexpr (STEP) {
    beam_bookkeeping(A, P, best);
  } else {
    if (tid < M) {
      const int64_t o = (int64_t)blockIdx.x * M + tid;
      A.out_scores[o] = best.value[tid];
      A.out_tokens[o] = best.token[tid];
      A.out_rows[o] = r0 + best.beam[tid];
    }
  }
}

namespace {

constexpr int BM_SLICE = BM_THREADS * 32;  // tokens of a workgroup

int64_t bm_slices(int64_t V) { return (V + 7 + BM_SLICE - 1) / BM_SLICE; }

int bm_run(BmArgs& a, const BmStep* step, int64_t prompts, int dtype, void* workspace, size_t bytes, hipStream_t stream,
           const std::string& w) {
  const int64_t rows = prompts * a.beams;
  a.S = (int)bm_slices(a.V);
  const size_t need = (size_t)(rows * a.S) * (8u * (size_t)a.M + 8u);
  if (!workspace || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))
    return fail(RWKV7MI_ESIZE, w + ": workspace missing, unaligned or smaller than rwkv7mi_beam_workspace_bytes");
  a.got = static_cast<uint64_t*>(workspace);
  a.sums = reinterpret_cast<float2*>(a.got + rows * a.S * a.M);
  const int rc = dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    constexpr int RUNS = 32 / (16 / (int)sizeof(T));
    hipLaunchKernelGGL((beam_slice_kernel<T, RUNS>), dim3((unsigned)a.S, (unsigned)rows), dim3(BM_THREADS), 0, stream, a);
    return check_launch("beam_slice_kernel");
  });
  if (rc) return rc;
  if (step)
    hipLaunchKernelGGL((beam_merge_kernel<1024, true>), dim3((unsigned)prompts), dim3(1024), 0, stream, a, *step);
  else
    hipLaunchKernelGGL((beam_merge_kernel<1024, false>), dim3((unsigned)prompts), dim3(1024), 0, stream, a, BmStep{});
  return check_launch("beam_merge_kernel");
}

int bm_check(const std::string& w, const void* x, int64_t prompts, int64_t beams, int64_t V, int64_t ldx, int dtype, int64_t M) {
  if (prompts < 0 || beams <= 0 || V <= 0 || ldx < 0 || M <= 0) return fail(RWKV7MI_EINVAL, w + ": bad shape");
  if (!valid_dtype(dtype)) return fail(RWKV7MI_EINVAL, w + ": bad dtype");
  if (M > BM_MOST || beams > BM_MOST)
    return fail(RWKV7MI_EINVAL, w + ": at most 128 beams and candidates of a prompt");
  if (V > INT32_MAX / 256) return fail(RWKV7MI_EINVAL, w + ": too large");
  if (reinterpret_cast<uintptr_t>(x) & (dtype == RWKV7MI_F32 ? 3 : 1)) return fail(RWKV7MI_EINVAL, w + ": unaligned logits");
  if (M > beams * V) return fail(RWKV7MI_EINVAL, w + ": more candidates than there are");
  if (prompts * beams > 65535) return fail(RWKV7MI_EINVAL, w + ": at most 65535 rows");
  return RWKV7MI_OK;
}

}  // namespace

}  // namespace rwkv7mi

using namespace rwkv7mi;

extern "C" size_t rwkv7mi_beam_workspace_bytes(int64_t rows, int64_t V, int64_t candidates) {
  if (rows <= 0 || V <= 0 || candidates <= 0) return 0;
  return (size_t)(rows * bm_slices(V)) * (8u * (size_t)candidates + 8u);
}

extern "C" int rwkv7mi_beam_select(const void* x, int64_t prompts, int64_t beams, int64_t V, int64_t ldx, int dtype,
                                   const float* scores, int normalized, int64_t candidates, float* out_scores,
                                   int64_t* out_tokens, int64_t* out_rows, void* workspace, size_t workspace_bytes,
                                   void* stream) {
  const std::string w("beam_select");
  if (int rc = bm_check(w, x, prompts, beams, V, ldx, dtype, candidates)) return rc;
  if (prompts == 0) return RWKV7MI_OK;
  if (!x || !scores || !out_scores || !out_tokens || !out_rows) return fail(RWKV7MI_EINVAL, w + ": null pointer");
  BmArgs a{x, ldx, (int)V, (int)beams, 0, (int)candidates, normalized, scores};
  a.out_scores = out_scores;
  a.out_tokens = out_tokens;
  a.out_rows = out_rows;
  return bm_run(a, nullptr, prompts, dtype, workspace, workspace_bytes, as_stream(stream), w);
}

extern "C" int rwkv7mi_beam_step(const void* x, int64_t prompts, int64_t beams, int64_t V, int64_t ldx, int dtype,
                                 int normalized, const int64_t* ends, int n_ends, double length_penalty,
                                 int early_stopping, int64_t pad, const rwkv7mi_beam_state* in,
                                 const rwkv7mi_beam_state* out, int64_t room, int64_t* next, int64_t* rows,
                                 void* workspace, size_t workspace_bytes, void* stream) {
  const std::string w("beam_step");
  if (n_ends < 0 || n_ends > BM_ENDS || (n_ends && !ends)) return fail(RWKV7MI_EINVAL, w + ": at most 8 end tokens");
  if (int rc = bm_check(w, x, prompts, beams, V, ldx, dtype, beams > BM_MOST ? beams : (1 + n_ends) * beams)) return rc;
  if (early_stopping < 0 || early_stopping > 2 || room <= 0 || room > INT32_MAX - 1)
    return fail(RWKV7MI_EINVAL, w + ": bad early_stopping or room");
  if (!(length_penalty == length_penalty)) return fail(RWKV7MI_EINVAL, w + ": length_penalty is NaN");
  if (prompts == 0) return RWKV7MI_OK;
  if (!x || !next || !rows || !in || !out) return fail(RWKV7MI_EINVAL, w + ": null pointer");
  BmStep p{};
  for (int side = 0; side < 2; ++side) {
    const rwkv7mi_beam_state* s = side ? out : in;
    if (!s->tokens || !s->lengths || !s->scores || !s->prompt_lengths || !s->finished_tokens || !s->finished_lengths ||
        !s->finished_scores || !s->done)
      return fail(RWKV7MI_EINVAL, w + ": null pointer in a state");
    (side ? p.out : p.in) = BmState{s->tokens, s->lengths, s->scores, s->prompt_lengths, s->finished_tokens,
                                    s->finished_lengths, s->finished_scores, s->done};
  }
  p.room = room;
  p.pad = pad;
  p.next = next;
  p.rows = rows;
  p.penalty = length_penalty;
  p.early = early_stopping;
  p.in_place = in->tokens == out->tokens;
  p.ends = n_ends;
  for (int e = 0; e < n_ends; ++e) p.end[e] = ends[e];
  BmArgs a{x, ldx, (int)V, (int)beams, 0, (int)((1 + n_ends) * beams), normalized, in->scores};
  return bm_run(a, &p, prompts, dtype, workspace, workspace_bytes, as_stream(stream), w);
}
