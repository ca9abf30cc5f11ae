// Beam search's step on the device: the best candidates of a prompt over its
// beams and the vocabulary, and what follows from them.
//
// For prompt b, beam k with running score s and logits x[0 .. V-1]:
//   value(k, t) = s + (x[t] - lse),  lse = m + log sum_t exp(x[t] - m)
// in 64 bits, rounded once to fp32 (close candidates are not equal for that); the
// exponentials and their sums over a slice are fp32, the slices' sums joined in 64
// bits.  The M best of the K V values, best
// first, equal ones by beam, then logit, then token.  A row that holds NaN or +inf, or whose score is
// one, is NaN throughout, and NaN ranks first, as in the argmax; a token of
// logit -inf, and every token of a row that is -inf throughout or whose score
// is, has the value -inf.
//
// beam_slice_kernel: one workgroup per slice of a row, one pass over the logits
// (aligned runs of 16 bytes, held in registers as they are): the slice's maximum and sum of exponentials (fp32, of
// exact differences from the maximum), and its M best logits (a row's score and
// lse do not change the order inside it).  The lanes' maxima give a bound: at
// least M values of the slice reach the M-th largest of them, found bit by bit
// with ballots, or a little less (16 more pass: fewer bits); the few runs that
// hold one go through LDS to the wave's lanes, and what reaches the bound is
// ranked by counting.  -inf is never gathered: a masked row costs no more than
// another.  Values in numbers that LDS does not hold (long ties) are drawn one by
// one instead.  Bound by memory and vector instructions together for many rows:
// 67 MB in 17.1 us, 3.9 TB/s, the vector units busy for 57% of the busy cycles;
// latency-bound for few (4.4 us for 4 rows).  (The least of the maxima of
// 16 groups of lanes as the bound, without the search: a selection of 64 x 8 rows
// 26.6 us against 24.9.)
//
// beam_merge_kernel: one workgroup per prompt joins the slices' sums to lse, in
// 64 bits, and selects among their K S M candidates the same way, the bound from
// the lists' heads; the step's bookkeeping (ends, hypotheses, places of the
// beams) follows in the same workgroup, two of its waves deciding without a
// barrier.  Latency-bound, a chain of short phases: 4.8 us for one prompt of 4
// beams, 7.8 for 64 of 8, 9 to 15 (by what reaches the bound) for 4 of 32 with 64
// candidates; as a step's 8.1 and 17.2 for the first two.
//
// Whole selections in a captured graph: 1 x 4 rows of 65536 fp16 logits 8.7 to
// 9.0 us, 64 x 8 24.0 (12.5 at the rate of a large copy), 4 x 32 fp32 25.8; steps of
// the first two 11.5 and 42.7, texts of 4096 tokens of room included in the second.
#include "common.h"

namespace rwkv7mi {

namespace {

constexpr int BM_THREADS = 256;
constexpr int BM_MERGE = 1024;    // lanes that join a prompt's slices
constexpr int BM_CAP = 1024;      // candidates that a workgroup gathers, whole 64s
constexpr int BM_WAVE_RUNS = 128; // runs of them that a wave gathers
constexpr int BM_RANKED = 320;    // of them ranked without a second bound
constexpr int BM_MOST = 128;      // candidates of a prompt
constexpr int BM_ENDS = 8;        // end tokens
constexpr int64_t BM_ROOM = 1 << 30;  // tokens of room (a copy's offsets, in steps of 512, are 32 bits wide)

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
  int* plan;  // [prompts][2 beams] where the texts of the rows and of the hypotheses come from, for
              // beam_texts_kernel (null: copied with the decision): a row of the prompt, -1 as it was
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

// the wave's maximum, in every lane (NaN counts as nothing)
__device__ __forceinline__ float bm_wave_max(float v) {
  v = fmaxf(v, dpp_row_ror<8>(v));
  v = fmaxf(v, dpp_row_ror<4>(v));
  v = fmaxf(v, dpp_row_ror<2>(v));
  v = fmaxf(v, dpp_row_ror<1>(v));
  return fmaxf(fmaxf(lane_f(v, 0), lane_f(v, 16)), fmaxf(lane_f(v, 32), lane_f(v, 48)));
}

// what the lanes of a wave wrote to LDS is there for the others
__device__ __forceinline__ void bm_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// the maximum and the total over the 16 lanes of a row, in each of them
__device__ __forceinline__ float bm_row_max(float v) {
  v = fmaxf(v, dpp_row_ror<8>(v));
  v = fmaxf(v, dpp_row_ror<4>(v));
  v = fmaxf(v, dpp_row_ror<2>(v));
  return fmaxf(v, dpp_row_ror<1>(v));
}
template <int N>
__device__ __forceinline__ double bm_turn(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, 0x120 + N, 0xF, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), 0x120 + N, 0xF, 0xF, false);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double bm_row_sum(double v) {
  v += bm_turn<8>(v);
  v += bm_turn<4>(v);
  v += bm_turn<2>(v);
  return v + bm_turn<1>(v);
}
// the total over the 16 lanes of a row, in each of them
__device__ __forceinline__ int bm_row_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x124, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x122, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x121, 0xF, 0xF, false);
  return v;
}

// A bound that at least M of the 64 Q keys in LDS reach, and no more than M + SLACK of them where bits
// LOW and up can tell (the largest such, bit by bit from the top); BM_NONE + 1 where fewer than M are
// above BM_NONE.  One wave.
template <int Q, int LOW>
__device__ __forceinline__ uint32_t bm_bound(const uint32_t* keys, int M) {
  constexpr int SLACK = 16;
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
    if (n >= M && n <= M + SLACK) break;
  }
  return max(t, BM_NONE + 1);
}

}  // namespace

namespace {

// element e of a run of 16 bytes
template <typename T>
__device__ __forceinline__ float bm_element(const uint32_t (&d)[4], int e) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(d[e]);
  } else {
    const uint32_t w = d[e / 2];
    return to_f32(__builtin_bit_cast(T, (uint16_t)(e & 1 ? w >> 16 : w & 0xffffu)));
  }
}

constexpr float BM_LOG2E = 1.44269504f;
// log2(e) times that element less m, to be exponentiated.  fp16: less base = fp32(log2(e) m), in one
// instruction (the product exact; what base was rounded by is put right in the sum); the others, whose
// products could overflow: the difference first.
template <typename T>
__device__ __forceinline__ float bm_less(const uint32_t (&d)[4], int e, float m, float base) {
  if constexpr (std::is_same<T, __half>::value) {
    float r;  // (the conversion inside)
    const uint32_t w = d[e / 2];
    if (e & 1)
      asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(BM_LOG2E), "v"(base));
    else
      asm("v_fma_mix_f32 %0, %1, %2, -%3 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(w), "v"(BM_LOG2E), "v"(base));
    return r;
  } else {
    return (bm_element<T>(d, e) - m) * BM_LOG2E;
  }
}

// the largest element of a run (NaN counts as nothing, or as the largest)
template <typename T>
__device__ __forceinline__ float bm_run_max(const uint32_t (&d)[4]) {
  if constexpr (std::is_same<T, __half>::value) {
    f16x2 h[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t w = d[q];
      h[q] = __builtin_bit_cast(f16x2, w);
    }
    const f16x2 t = __builtin_elementwise_max(__builtin_elementwise_max(h[0], h[1]), __builtin_elementwise_max(h[2], h[3]));
    return fmaxf((float)t[0], (float)t[1]);
  } else {
    float t = bm_element<T>(d, 0);
#pragma unroll
    for (int e = 1; e < 16 / (int)sizeof(T); ++e) t = fmaxf(t, bm_element<T>(d, e));
    return t;
  }
}

}  // namespace

// RUNS 16-byte runs a lane, kept as they are in memory.
template <typename T, int RUNS>
__global__ __launch_bounds__(BM_THREADS) void beam_slice_kernel(const BmArgs A) {
  constexpr int E = 16 / (int)sizeof(T), SLICE = BM_THREADS * RUNS * E, WAVES = BM_THREADS / 64;
  constexpr int LOW = std::is_same<T, __half>::value ? 13 : sizeof(T) == 2 ? 16 : 0;  // bits that T's values have
  __shared__ uint64_t got[BM_CAP];
  __shared__ uint32_t top[BM_THREADS];
  __shared__ uint32_t bound;
  __shared__ float wave_top[WAVES], wave_sums[WAVES];
  __shared__ u32x4 run[WAVES][BM_WAVE_RUNS];
  __shared__ uint16_t run_at[WAVES][BM_WAVE_RUNS];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int beam = (int)blockIdx.y;
  const int64_t row = (int64_t)blockIdx.z * A.beams + beam;
  const T* x = static_cast<const T*>(A.x) + row * A.ldx;
  const int shift = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int c0 = (int)blockIdx.x * SLICE - shift;  // the slice's first token (before the row in the first slice)
  const int t0 = c0 + E * tid;
  // aligned units of 16 bytes that hold a token of the row (no such unit crosses a page), all at once; what
  // of them lies outside the row is nothing
  const __amdgpu_buffer_rsrc_t mem = make_rsrc(x - shift, ((uint32_t)(shift + A.V) * (uint32_t)sizeof(T) + 15u) & ~15u);
  uint32_t d[RUNS][4];
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int i = t0 + E * BM_THREADS * u;
    const u32x4 w = buf_ld16(mem, (uint32_t)(i + shift) * (uint32_t)sizeof(T));
#pragma unroll
    for (int q = 0; q < 4; ++q) d[u][q] = w[q];
  }
  if (c0 < 0 || c0 + SLICE > A.V) {
    constexpr uint32_t NOTHING = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
      const int i = t0 + E * BM_THREADS * u;
      if (i >= 0 && i + E <= A.V) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const bool in = i + e >= 0 && i + e < A.V;
        const uint32_t mask = sizeof(T) == 4 ? ~0u : 0xffffu << (16 * (e & 1));
        uint32_t& w = d[u][e * (int)sizeof(T) / 4];
        w = in ? w : (w & ~mask) | (NOTHING & mask);
      }
    }
  }
  float run_best[RUNS], best = -__builtin_inff();
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    run_best[u] = bm_run_max<T>(d[u]);
    best = fmaxf(best, run_best[u]);
  }
  if (tid == 0) count = 0;
#pragma unroll
  for (int i = 0; i < BM_CAP / BM_THREADS; ++i) got[BM_THREADS * i + tid] = 0;
  top[tid] = bm_key(best);
  best = bm_wave_max(best);
  if (lane == 0) wave_top[wave] = best;
  __syncthreads();
  float m = wave_top[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) m = fmaxf(m, wave_top[w]);
  if (wave == 0) {
    const uint32_t t = bm_bound<WAVES, LOW>(top, A.M);
    if (tid == 0) bound = t;
  }
  // NaN and +inf make the sum NaN (a slice of -inf and NaN alone: asked for)
  const float base = m * BM_LOG2E;
  float s = 0.f;
  if (m > -__builtin_inff()) {
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
#pragma unroll
      for (int e = 0; e < E; ++e) s += __builtin_amdgcn_exp2f(bm_less<T>(d[u], e, m, base));
      __builtin_amdgcn_sched_barrier(0);  // (one run's exponentials at a time: registers)
    }
  } else {
#pragma unroll
    for (int u = 0; u < RUNS; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = bm_element<T>(d[u], e);
        s = v != v ? v : s;
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  s = wave_sum(s);
  if (lane == 0) wave_sums[wave] = s;
  __syncthreads();
  const float reach = bm_value(bound);
  const int64_t slice = row * A.S + blockIdx.x;
  uint64_t* out = A.got + slice * A.M;
  // the runs that hold one that reaches go to LDS as they are, and the wave's lanes take their elements:
  // no lane waits for what another one found
  int held = 0;
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const bool hit = run_best[u] >= reach;
    const uint64_t hits = __ballot(hit);
    const int p = held + __popcll(hits & ((1ull << lane) - 1));
    if (hit && p < BM_WAVE_RUNS) {
      run[wave][p] = u32x4{d[u][0], d[u][1], d[u][2], d[u][3]};
      run_at[wave][p] = (uint16_t)(BM_THREADS * u + tid);
    }
    held += __popcll(hits);
  }
  bm_wave_sync();
  if (held > BM_WAVE_RUNS) {  // (drawn one by one)
    if (lane == 0) atomicAdd(&count, BM_CAP + 1);
  } else {
    for (int i = lane / E; i < held; i += 64 / E) {
      const float v = to_f32(reinterpret_cast<const T*>(&run[wave][i])[lane % E]);
      if (v >= reach) {
        const int p = atomicAdd(&count, 1);
        if (p < BM_CAP) got[p] = (uint64_t)bm_key(v) << 32 | (uint32_t) ~(c0 + E * run_at[wave][i] + lane % E);
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) sum += wave_sums[w];
    if (std::is_same<T, __half>::value && m > -__builtin_inff()) sum *= __builtin_amdgcn_exp2f(fmaf(-m, BM_LOG2E, base));
    A.sums[slice] = make_float2(m, sum);
  }
  const int n = count;
  if (n <= BM_CAP) {
    for (int i = tid >> 4; i < n; i += BM_THREADS / 16) {  // 16 lanes a candidate
      const uint64_t k = got[i];
      int r = 0;
      for (int j = tid & 15; j < n; j += 64) r += (got[j] > k) + (got[j + 16] > k) + (got[j + 32] > k) + (got[j + 48] > k);
      r = bm_row_sum(r);
      if (r < A.M && (tid & 15) == 0) out[r] = bm_pack((uint32_t)(k >> 32), beam, (int)~(uint32_t)k);
    }
    for (int r = n + tid; r < A.M; r += BM_THREADS) out[r] = 0;
    return;
  }
  // too many reach the bound: M times the best below the last
  uint64_t last = ~0ull;
  for (int r = 0; r < A.M; ++r) {
    uint64_t k = 0;
    int t = t0;
#pragma unroll
    for (int u = 0; u < RUNS; ++u) {
      asm volatile("" : "+v"(t));
#pragma unroll
      for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(d[u][q]));  // (converted anew each time: registers)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = bm_element<T>(d[u], e);
        const uint64_t c = (uint64_t)bm_key(v) << 32 | (uint32_t) ~(t + E * BM_THREADS * u + e);
        if (v >= reach && c < last && c > k) k = c;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const uint64_t c = __shfl_xor((unsigned long long)k, o, 64);
      k = max(k, c);
    }
    __syncthreads();
    if (lane == 0) got[wave] = k;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) k = max(k, got[w]);
    last = k;
    if (tid == 0) out[r] = bm_pack((uint32_t)(k >> 32), beam, (int)~(uint32_t)k);
  }
}

namespace {

struct BmBest {  // a prompt's candidates, best first
  float value[BM_MOST];
  int token[BM_MOST], beam[BM_MOST];
};

struct BmBook {  // what two waves decide and all copy by
  int live[BM_MOST], place[BM_MOST], taken[BM_MOST];  // taken: the hypothesis of a slot, -1: as before
  float hyp[BM_MOST], old[BM_MOST];
  int old_length[BM_MOST];
  int list[BM_MOST], owner[BM_MOST], newcomer[BM_MOST];
  double span;
};

template <typename V>
__device__ __forceinline__ void bm_copy_units(V* dst, const V* src, int n) {
  int i = threadIdx.x & 63;
  for (; i + 448 < n; i += 512) {
    V t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) t[u] = src[i + 64 * u];
#pragma unroll
    for (int u = 0; u < 8; ++u) dst[i + 64 * u] = t[u];
  }
  V t[8] = {};
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (i + 64 * u < n) t[u] = src[i + 64 * u];
#pragma unroll
  for (int u = 0; u < 8; ++u)
    if (i + 64 * u < n) dst[i + 64 * u] = t[u];
}
// a row of n tokens by one wave, eight loads in flight, of two tokens where the rows' alignment allows it
__device__ __forceinline__ void bm_copy(int64_t* dst, const int64_t* src, int n) {
  if (((reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(src)) & 15) == 0) {
    bm_copy_units(reinterpret_cast<u32x4*>(dst), reinterpret_cast<const u32x4*>(src), n / 2);
    if (n & 1 && (threadIdx.x & 63) == 0) dst[n - 1] = src[n - 1];
  } else {
    bm_copy_units(dst, src, n);
  }
}

}  // namespace

// whether candidate r ends its text
__device__ __forceinline__ bool bm_ends(const BmStep& P, const BmBest& best, int r) {
  bool end = false;
  for (int e = 0; e < P.ends; ++e) end |= best.token[r] == P.end[e];
  return end && best.value[r] > -__builtin_inff();
}

// One wave: which candidates live on, and where.
__device__ __forceinline__ void beam_live(const BmArgs& A, const BmStep& P, const BmBest& best, BmBook& k) {
  const int lane = threadIdx.x & 63, K = A.beams;
  const uint64_t below = (1ull << lane) - 1;
  // the first K that do not end
  for (int r0 = 0, lives = 0; r0 < A.M && lives < K; r0 += 64) {
    const int r = r0 + lane;
    const bool stays = r < A.M && !bm_ends(P, best, r);
    const uint64_t on = __ballot(stays);
    const int rank = lives + __popcll(on & below);
    if (stays && rank < K) k.live[rank] = r;
    lives += __popcll(on);
  }
  for (int r = lane; r < K; r += 64) k.owner[r] = K;
  bm_wave_sync();
  // a beam's first child keeps its row, the others take the rows that are left
  for (int r = lane; r < K; r += 64) atomicMin(&k.owner[best.beam[k.live[r]]], r);
  bm_wave_sync();
  for (int r0 = 0, spare = 0; r0 < K; r0 += 64) {
    const int r = r0 + lane;
    const uint64_t free = __ballot(r < K && k.owner[r] == K);
    if (free >> lane & 1) k.list[spare + __popcll(free & below)] = r;
    spare += __popcll(free);
  }
  bm_wave_sync();
  for (int r0 = 0, twins = 0; r0 < K; r0 += 64) {
    const int r = r0 + lane, beam = r < K ? best.beam[k.live[r]] : 0;
    const uint64_t twin = __ballot(r < K && k.owner[beam] != r);
    if (r < K) k.place[r] = twin >> lane & 1 ? k.list[twins + __popcll(twin & below)] : beam;
    twins += __popcll(twin);
  }
}

// Another wave: the K best of the hypotheses so far and of those that end here, earlier ones first.
__device__ __forceinline__ void beam_end(const BmArgs& A, const BmStep& P, const BmBest& best, BmBook& k, bool last) {
  const int lane = threadIdx.x & 63, K = A.beams;
  const uint64_t below = (1ull << lane) - 1;
  bool any = false;
  for (int r = lane; r < K; r += 64) {
    const float v = best.value[r];
    const bool ends = bm_ends(P, best, r) || (last && v > -__builtin_inff());
    const float h = ends ? (float)((double)v / k.span) : -__builtin_inff();
    k.hyp[r] = h;
    k.taken[r] = -1;
    any |= h > -__builtin_inff();
  }
  if (!__any(any)) return;
  bm_wave_sync();
  uint64_t kept[2] = {0, 0};
  int newcomers = 0;
  for (int q = 0; q < 2 && 64 * q < K; ++q) {
    const int r = 64 * q + lane;
    const float o = r < K ? k.old[r] : 0.f, h = r < K ? k.hyp[r] : -__builtin_inff();
    int ro = r < K ? 0 : K, rh = 0;
#pragma unroll 4
    for (int j = 0; j < K; ++j) {
      const float oj = k.old[j], hj = k.hyp[j];
      ro += ((oj > o) | ((oj == o) & (j < r))) + (hj > o);
      rh += (oj >= h) + ((hj > h) | ((hj == h) & (j < r)));
    }
    kept[q] = __ballot(ro < K);
    const uint64_t in = __ballot(h > -__builtin_inff() && rh < K);
    if (in >> lane & 1) k.newcomer[newcomers + __popcll(in & below)] = r;
    newcomers += __popcll(in);
  }
  bm_wave_sync();
  for (int q = 0, gone = 0; q < 2 && 64 * q < K; ++q) {
    const int r = 64 * q + lane;
    const uint64_t go = __ballot(r < K && !(kept[q] >> lane & 1));
    const int at = gone + __popcll(go & below);
    if ((go >> lane & 1) && at < newcomers) k.taken[r] = k.newcomer[at];
    gone += __popcll(go);
  }
}

// All waves: the step behind the selection.  was, len and prompt are the prompt's.
__device__ __forceinline__ void beam_bookkeeping(const BmArgs& A, const BmStep& P, const BmBest& best, BmBook& book, bool was,
                                                 int len, int prompt) {
  const int tid = threadIdx.x, K = A.beams, waves = blockDim.x >> 6, wave = tid >> 6;
  const int64_t b = blockIdx.x, r0 = b * K;
  if (was || len < 0 || len >= P.room) {  // (no room: nothing can follow)
    if (P.plan && tid < 2 * K) P.plan[2 * r0 + tid] = -1;
    if (!P.in_place && !P.plan)
      for (int j = wave; j < 2 * K; j += waves) {
        const int64_t at = (r0 + (j >> 1)) * P.room;
        if (j & 1)
          bm_copy(P.out.finished_tokens + at, P.in.finished_tokens + at, book.old_length[j >> 1]);
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
  const bool last = len + 1 >= P.room;  // the rows are full behind this token: all texts end
  if (wave == 0) beam_live(A, P, best, book);
  if (wave == 1) beam_end(A, P, best, book, last);
  __syncthreads();
  const int *live = book.live, *place = book.place, *taken = book.taken;
  const float *hyp = book.hyp, *old = book.old;
  if (P.plan && tid < K) {
    P.plan[2 * r0 + place[tid]] = best.beam[live[tid]];
    P.plan[2 * r0 + K + tid] = taken[tid] >= 0 ? best.beam[taken[tid]] : -1;
  }
  // the texts: a wave a row; hypotheses first: in place, a row whose only child ended may be taken
  for (int k = wave; k < K && !P.plan; k += waves) {
    const int h = taken[k];
    int64_t* dst = P.out.finished_tokens + (r0 + k) * P.room;
    if (h >= 0)
      bm_copy(dst, P.in.tokens + (r0 + best.beam[h]) * P.room, len);
    else if (!P.in_place)
      bm_copy(dst, P.in.finished_tokens + (r0 + k) * P.room, book.old_length[k]);
  }
  if (P.in_place) __syncthreads();
  for (int i = P.in_place ? wave : (wave + waves - K % waves) % waves; i < K && !P.plan; i += waves) {
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
  if (wave == waves - 1) {
    float worst = __builtin_inff();
    for (int k = tid & 63; k < K; k += 64) worst = fminf(worst, taken[k] >= 0 ? hyp[taken[k]] : old[k]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) worst = fminf(worst, __shfl_xor(worst, o, 64));
    if ((tid & 63) == 0) {
      // early 0: at the present length; 1: as soon as there are K hypotheses; 2: at the length that helps most
      const double ahead = P.early == 2 && P.penalty > 0 ? pow((double)max(P.room - prompt, (int64_t)1), P.penalty) : book.span;
      const bool over = P.early == 1 ? worst > -__builtin_inff()
                                     : !((float)((double)best.value[live[0]] / ahead) > worst);
      P.out.done[b] = over || last;
      P.out.prompt_lengths[b] = prompt;
    }
  }
}

template <bool STEP>
__global__ __launch_bounds__(BM_MERGE) void beam_merge_kernel(const BmArgs A, const BmStep P) {
  constexpr int NT = BM_MERGE;
  constexpr int HOLD = 4;  // candidates that a lane keeps; further ones are read twice
  __shared__ uint64_t got[BM_CAP];
  __shared__ uint64_t got_at[BM_CAP];  // what decides where values are equal (bm_place), the least first
  __shared__ uint32_t keys[BM_CAP];  // of a sample of the candidates, then of those gathered
  __shared__ double lse[BM_MOST];
  __shared__ float score[BM_MOST];
  __shared__ int by_kind[BM_MOST];  // the rows of NaN, in order; then the others
  __shared__ bool odd[BM_MOST];      // rows of NaN
  __shared__ float offset[BM_MOST];  // score - lse in fp32
  __shared__ uint32_t bound;
  __shared__ int count;
  __shared__ BmBest best;
  __shared__ BmBook book;
  const int tid = threadIdx.x, lane = tid & 63, K = A.beams, M = A.M;
  const int64_t r0 = (int64_t)blockIdx.x * K;
  const int L = K * A.S, N = L * M;  // lists, candidates
  const uint64_t* list = A.got + r0 * A.S * M;
  // candidates by chunks: the next 2^chunk of every list (they are in order), as many as fit HOLD a lane
  int chunk = 0;
  while (1 << chunk < M && (L << (chunk + 1)) <= NT * HOLD) ++chunk;
  const int wide = L << chunk;
  const auto at = [&](int j, int rank0) {  // candidate j of a chunk
    const int r = rank0 + (j & ((1 << chunk) - 1));
    return j < wide && r < M ? list[(int64_t)(j >> chunk) * M + r] : 0;
  };
  // a sample of 64 or 256 gives the bound: the best of every list and, where lists are few, the next ones.
  // (64 cost half the time for a bound that lets a few more through: M of them have to reach it)
  const int sample = M <= 24 ? 64 : 256;
  // everything that is read is on its way while lse is formed
  const int row = tid >> 4, part0 = tid & 15;  // 16 lanes a row
  float own = row < K ? A.scores[r0 + row] : 0.f;
  const auto sums_of = [&](int k, int j) {
    return k < K && j < A.S ? A.sums[(r0 + k) * A.S + j] : make_float2(-__builtin_inff(), 0.f);
  };
  float2 sums = sums_of(row, part0);
  uint64_t held[HOLD], head = 0;
  if (tid < sample && L <= sample && tid / L < M) head = list[(tid % L) * M + tid / L];
#pragma unroll
  for (int i = 0; i < HOLD; ++i) held[i] = at(tid + NT * i, 0);
  bool was = false;
  int len = 0, prompt = 0;
  if constexpr (STEP) {
    was = P.in.done[blockIdx.x];
    len = P.in.lengths[r0];
    prompt = P.in.prompt_lengths[blockIdx.x];
    const int k = tid - (NT - BM_MOST);  // (the last waves have no row of sums, as a rule)
    if (k >= 0 && k < K) {
      book.old[k] = P.in.finished_scores[r0 + k];
      book.old_length[k] = min(max(P.in.finished_lengths[r0 + k], 0), (int)P.room);
    }
    if (tid == NT - 1) {
      const double gen = max(len + 1 - prompt, 1);
      book.span = P.penalty == 1.0 ? gen : pow(gen, P.penalty);
    }
  }
  if (tid == 0) count = 0;
  got[tid] = 0;
  if (tid < BM_MOST) {  // (what a workspace that another call writes leaves unset points into the prompt too)
    best.value[tid] = -__builtin_inff();
    best.beam[tid] = best.token[tid] = 0;
    if constexpr (STEP) book.live[tid] = 0;
  }
  for (int k = row; k < K; k += NT / 16) {
    if (k != row) {
      own = A.scores[r0 + k];
      sums = sums_of(k, part0);
    }
    float m = sums.x;
    for (int j = part0 + 16; j < A.S; j += 16) m = fmaxf(m, sums_of(k, j).x);
    m = bm_row_max(m);
    const auto part = [&](float2 q) {
      return q.x > -__builtin_inff() ? (double)q.y * exp((double)q.x - (double)m) : (double)q.y;
    };
    double s = part(sums);
    for (int j = part0 + 16; j < A.S; j += 16) s += part(sums_of(k, j));
    s = bm_row_sum(s);
    const bool nan = s != s || !(own < __builtin_inff());
    if (part0 == 0) {
      const double l = A.normalized || nan || !(s > 0.0) ? 0.0 : (double)m + log(s);
      lse[k] = l;
      odd[k] = nan;
      score[k] = nan ? -__builtin_inff() : own;  // (nothing to choose by value)
      // (finite where own is: what it is cut off by is covered by the allowance in gather, or that is infinite)
      offset[k] = nan || own == -__builtin_inff() ? -__builtin_inff()
                                                  : fminf(fmaxf((float)((double)own - l), -__FLT_MAX__), __FLT_MAX__);
    }
  }
  __syncthreads();
  const uint64_t nan0 = __ballot(lane < K && odd[lane & (BM_MOST - 1)]);
  const uint64_t nan1 = K > 64 ? __ballot(lane + 64 < K && odd[lane + 64]) : 0;
  const int bad = __popcll(nan0) + __popcll(nan1);
  const int first = (int)min((int64_t)bad * A.V, (int64_t)M);  // NaN ranks first
  const int want = M - first;
  const auto value = [&](uint64_t c) {  // -inf: nothing to choose
    const int k = (int)(c >> 23 & 0x7f);
    if ((uint32_t)(c >> 32) <= BM_NONE) return -__builtin_inf();
    return fmax((double)score[k] + ((double)bm_value((uint32_t)(c >> 32)) - lse[k]), -__builtin_inf());
  };
  if (tid < sample) {
    uint32_t mine = bm_key((float)value(head));
    if (L > sample)
      for (int l = tid; l < L; l += sample) mine = max(mine, bm_key((float)value(list[(int64_t)l * M])));
    keys[tid] = mine;
  }
  __syncthreads();
  if (tid < 64) {
    const uint32_t t = sample == 64 ? bm_bound<1, 0>(keys, max(want, 1)) : bm_bound<4, 0>(keys, max(want, 1));
    if (tid == 0) bound = t;
  }
  __syncthreads();
  uint32_t at_least = bound;
  float reach = bm_value(at_least);
  const auto gather = [&](uint64_t c) {  // whether it reaches the bound
    const float l = bm_value((uint32_t)(c >> 32)), o = offset[c >> 23 & 0x7f];
    // (fp32, less than four roundings off, and no bound where it is not finite; false for -inf and what is not there)
    if (l + o + 0x1p-21f * (fabsf(l) + fabsf(o)) < reach || o == -__builtin_inff() || (uint32_t)(c >> 32) <= BM_NONE)
      return false;
    const double v = value(c);
    if (bm_key((float)v) < at_least) return false;
    const int p = atomicAdd(&count, 1);
    if (p < BM_CAP) got[p] = bm_key(v), got_at[p] = bm_place(c);
    return true;
  };
  int n;
  for (;;) {
    // further chunks only behind lists whose last candidate so far reaches the bound
    const int last = (1 << chunk) - 1;
    bool more = false;
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
      if (NT * i < wide) more |= gather(held[i]) && ((tid + NT * i) & last) == last;
    for (int j = tid + NT * HOLD; j < wide; j += NT) more |= gather(at(j, 0)) && (j & last) == last;
    for (int rank = 1 << chunk; rank < M && __syncthreads_or(more); rank += 1 << chunk) {
      more = false;
      for (int j = tid; j < wide; j += NT) more |= gather(at(j, rank)) && (j & last) == last;
    }
    __syncthreads();
    n = count;
    if (n <= BM_CAP) break;
    // too many, as where the best beams have most of the best candidates: those gathered, whichever they
    // are, give a better bound (unless they are equal: then they are drawn one by one)
    keys[tid] = bm_key((float)bm_value(got[tid]));
    __syncthreads();
    if (tid < 64) {
      const uint32_t t = bm_bound<BM_CAP / 64, 0>(keys, max(want, 1));
      if (tid == 0) bound = t, count = 0;
    }
    got[tid] = 0;
    __syncthreads();
    if (bound <= at_least) break;
    at_least = bound;
    reach = bm_value(at_least);
  }
  // (ranking by counting reads n entries for each: many are cut down by a bound of their own first)
  if (n > BM_RANKED && n <= BM_CAP) {
    uint64_t k = 0, p = 0;
    if (tid < n) k = got[tid], p = got_at[tid];
    const uint32_t key = tid < n ? bm_key((float)bm_value(k)) : 0u;
    keys[tid] = key;
    __syncthreads();
    got[tid] = 0;
    if (tid < 64) {
      const uint32_t t = bm_bound<BM_CAP / 64, 0>(keys, max(want, 1));
      if (tid == 0) bound = t, count = 0;
    }
    __syncthreads();
    if (key >= bound) {
      const int q = atomicAdd(&count, 1);
      got[q] = k, got_at[q] = p;
    }
    __syncthreads();
    n = count;
  }
  const auto put = [&](int r, float v, int beam, int token) {
    best.value[r] = v;
    best.beam[r] = min(beam, K - 1);
    best.token[r] = token;
  };
  if (n <= BM_CAP) {
    for (int i = tid >> 4; i < n; i += NT / 16) {  // 16 lanes a candidate
      const uint64_t k = got[i], at = got_at[i];
      int r = 0, same = 0;
      for (int j = tid & 15; j < n; j += 64) {  // (zeros behind the n)
        const uint64_t c0 = got[j], c1 = got[j + 16], c2 = got[j + 32], c3 = got[j + 48];
        r += (c0 > k) + (c1 > k) + (c2 > k) + (c3 > k);
        same += (c0 == k) + (c1 == k) + (c2 == k) + (c3 == k);
      }
      if (bm_row_sum(same) > 1)
        for (int j = tid & 15; j < n; j += 16) r += got[j] == k && got_at[j] < at;
      r = bm_row_sum(r);
      if (r < want && (tid & 15) == 0) put(first + r, (float)bm_value(k), bm_beam(at), bm_token(at));
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
  const int found = min(n, want);
  if (first || found < want) {
    // the rows of NaN give their tokens, and behind what can be chosen the others their -inf ones, both
    // by index: M values are there
    if (tid < K) {
      int q = 0;
      for (int j = 0; j < tid; ++j) q += odd[j] == odd[tid];
      by_kind[odd[tid] ? q : bad + q] = tid;
    }
    __syncthreads();
    if (tid < first) put(tid, __builtin_nanf(""), by_kind[tid / A.V], tid % A.V);
    if (found < want && tid < 64) {
      int r = first + found;
      for (int j0 = 0; r < M; j0 += 64) {
        const int j = j0 + lane, kind = bad + j / A.V;
        const bool there = kind < K;
        const int beam = there ? by_kind[kind] : 0, token = j % A.V;
        bool free = there;
        for (int i = 0; i < found && free; ++i) free = best.beam[first + i] != beam || best.token[first + i] != token;
        const uint64_t f = __ballot(free);
        const int p = r + __popcll(f & ((1ull << lane) - 1));
        if (free && p < M) put(p, -__builtin_inff(), beam, token);
        r += __popcll(f);
        if (!__any(there)) break;
      }
    }
  }
  __syncthreads();
  if constexpr (STEP) {
    beam_bookkeeping(A, P, best, book, was, len, prompt);
  } else {
    if (tid < M) {
      const int64_t o = (int64_t)blockIdx.x * M + tid;
      A.out_scores[o] = best.value[tid];
      A.out_tokens[o] = best.token[tid];
      A.out_rows[o] = r0 + best.beam[tid];
    }
  }
}

// The texts of a step into another state: one workgroup a row or hypothesis.  (The step's own
// workgroups, one a prompt, leave most of the card idle.  Steps over 8192 logits with this launch and
// with the copies in the step's: 1 x 32 texts of 1024 tokens of room 23.3 us and 27.5, 1 x 32 of 4096
// 24.0 and 40.3, 64 x 8 of 4096 25.7 and 26.9; 1 x 4 of 4096 13.6 and 12.9, 64 x 8 of 500 19.7 and 17.6.)
__global__ __launch_bounds__(256) void beam_texts_kernel(const BmStep P, int beams) {
  const int64_t b = blockIdx.y, row = b * beams + blockIdx.x % beams;
  const bool finished = (int)blockIdx.x >= beams;
  const int from = min(P.plan[2 * b * beams + blockIdx.x], beams - 1), room = (int)P.room;
  const int64_t* src = (finished && from < 0 ? P.in.finished_tokens : P.in.tokens) + (from < 0 ? row : b * beams + from) * P.room;
  int n = finished && from < 0 ? P.in.finished_lengths[row] : P.in.lengths[b * beams];
  n = min(max(n, 0), room);
  int64_t* dst = (finished ? P.out.finished_tokens : P.out.tokens) + row * P.room;
  // (a wave takes a run of whole 16-byte units)
  const int part = ((n + 3) / 4 + 1) & ~1, at = min((int)(threadIdx.x >> 6) * part, n);
  bm_copy(dst + at, src + at, min(part, n - at));
}

namespace {

int64_t bm_slice(int dtype, int runs) { return (int64_t)BM_THREADS * runs * (dtype == RWKV7MI_F32 ? 4 : 8); }
int64_t bm_slices(int64_t V, int dtype, int runs) { return (V + bm_slice(dtype, runs) - 1) / bm_slice(dtype, runs); }

// Runs of a lane: 8, whose slices share the bound and the ranking among the most logits, where there are
// logits for 512 such workgroups, 4 down to 128 and 2 below, which fill the card sooner.  us of a selection
// with 2, 4, 8 runs, rows of 65536 logits (the rule takes 2 below 32 rows, 4 below 128, 8 from there; of fp32
// below 16 and 64):
//   rows      4              32              128               256               512
//   fp16  8.7 9.0 9.6   9.7 9.8 10.2   14.5 13.7 13.9   18.8 18.5 17.3   27.0 22.3 21.6
//   bf16  8.9 9.3 10.5  9.7 9.7 10.6   15.4 14.6 14.6   19.9 20.6 18.1   28.0 24.2 23.8
//   fp32  9.4 8.8 9.5  10.4 9.6 9.9    18.5 15.7 15.8   25.6 20.4 20.6   42.4 31.9 32.7
// (It was fitted to fp16.  fp32 would take 4 runs throughout: 1 to 8% less.)
int bm_runs(int64_t rows, int64_t V, int dtype) {
  const int64_t logits = rows * V, unit = bm_slice(dtype, 8);
  return logits >= 512 * unit ? 8 : logits >= 128 * unit ? 4 : 2;
}

constexpr int64_t BM_TEXTS = 1 << 15;  // tokens of room a prompt from which a launch of their own copies the texts

int bm_run(BmArgs& a, BmStep* step, int64_t prompts, int dtype, void* workspace, size_t bytes, hipStream_t stream,
           const std::string& w) {
  const int64_t rows = prompts * a.beams;
  // (a row starts up to 7 elements behind a boundary)
  const bool straight = !(reinterpret_cast<uintptr_t>(a.x) & 15) &&
                        (rows == 1 || a.ldx * (dtype == RWKV7MI_F32 ? 4 : 2) % 16 == 0);
  const int64_t width = a.V + (straight ? 0 : 7);
  const int runs = bm_runs(rows, a.V, dtype);
  a.S = (int)bm_slices(width, dtype, runs);
  const size_t need = (size_t)(rows * a.S) * (8u * (size_t)a.M + 8u) + 8u * (size_t)rows;
  if (!workspace || bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7))
    return fail(RWKV7MI_ESIZE, w + ": workspace missing, unaligned or smaller than rwkv7mi_beam_workspace_bytes");
  a.got = static_cast<uint64_t*>(workspace);
  a.sums = reinterpret_cast<float2*>(a.got + rows * a.S * a.M);
  const int rc = dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const dim3 grid((unsigned)a.S, (unsigned)a.beams, (unsigned)prompts);
    if (runs == 8)
      hipLaunchKernelGGL((beam_slice_kernel<T, 8>), grid, dim3(BM_THREADS), 0, stream, a);
    else if (runs == 4)
      hipLaunchKernelGGL((beam_slice_kernel<T, 4>), grid, dim3(BM_THREADS), 0, stream, a);
    else
      hipLaunchKernelGGL((beam_slice_kernel<T, 2>), grid, dim3(BM_THREADS), 0, stream, a);
    return check_launch("beam_slice_kernel");
  });
  if (rc) return rc;
  if (!step) {
    hipLaunchKernelGGL(beam_merge_kernel<false>, dim3((unsigned)prompts), dim3(BM_MERGE), 0, stream, a, BmStep{});
    return check_launch("beam_merge_kernel");
  }
  if (!step->in_place && a.beams * step->room >= BM_TEXTS) step->plan = reinterpret_cast<int*>(a.sums + rows * a.S);
  hipLaunchKernelGGL(beam_merge_kernel<true>, dim3((unsigned)prompts), dim3(BM_MERGE), 0, stream, a, *step);
  if (step->plan) {
    if (const int e = check_launch("beam_merge_kernel")) return e;
    hipLaunchKernelGGL(beam_texts_kernel, dim3(2u * (unsigned)a.beams, (unsigned)prompts), dim3(256), 0, stream, *step, a.beams);
    return check_launch("beam_texts_kernel");
  }
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
  if (prompts > 65535 / beams) return fail(RWKV7MI_EINVAL, w + ": at most 65535 rows");
  return RWKV7MI_OK;
}

}  // namespace

}  // namespace rwkv7mi

using namespace rwkv7mi;

extern "C" size_t rwkv7mi_beam_workspace_bytes(int64_t rows, int64_t V, int64_t candidates) {
  if (rows <= 0 || V <= 0 || candidates <= 0) return 0;
  return (size_t)(rows * bm_slices(V + 7, RWKV7MI_F32, 2)) * (8u * (size_t)candidates + 8u) + 8u * (size_t)rows;
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
  if (early_stopping < 0 || early_stopping > 2 || room <= 0 || room > BM_ROOM)
    return fail(RWKV7MI_EINVAL, w + ": bad early_stopping, or a room outside 1 .. 2^30");
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
