// Products with an MXFP4 weight: y = epilogue(x W^T + bias), fp16 / bf16 rows
// x, or the same rows quantised to MXFP4 on the way.
//
// mx4_rows_kernel: a workgroup of NW waves computes 16 rows x 16 outputs; the
// waves share K, and their fp32 sums meet in LDS in wave order.  A wave advances
// 128 inputs (four blocks) a step: lane n + 16 q holds block q of output n, 16
// bytes of codes and one scale byte, which is the operand of
//  * one v_mfma_scale_f32_16x16x128_f8f6f4 where x is MXFP4 too, or
//  * four v_mfma_f32_16x16x32 where x is 16-bit: MFMA j takes inputs 8 j .. +7
//    of every lane's block, and so do the rows of x.
// bf16 holds a scaled code exactly.  fp16 does not for every scale, so there a
// step's codes are scaled relative to the largest of its four scales and the
// step's sums by that one's factor (mx4_common.h).
#include <algorithm>

#include "mx4_common.h"

namespace rwkv7mi {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 mx4_operand(u32x4 v) {
  return (i32x8){(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}

// exponent bytes of the four blocks of one step, block q in byte q; blocks past
// the row read 0.  WHOLE: I % 128 == 0 (a step's bytes are an aligned dword).
template <bool WHOLE>
__device__ __forceinline__ uint32_t mx4_exps(const uint8_t* row, int b, int nb) {
  if constexpr (WHOLE) return *reinterpret_cast<const uint32_t*>(row + b);
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (b + i < nb) v |= (uint32_t)row[b + i] << (8 * i);
  return v;
}

__device__ __forceinline__ uint32_t max4(uint32_t v) {
  return max(max(v & 255u, (v >> 8) & 255u), max((v >> 16) & 255u, v >> 24));
}

}  // namespace

template <typename T, bool A4, bool WHOLE>
__global__ __launch_bounds__(1024) void mx4_rows_kernel(const Mx4Batch B) {
  using V = typename Mx4Types<T>::V;
  constexpr bool F16 = std::is_same<T, __half>::value && !A4;
  const Mx4Prob& P = B.p[blockIdx.z];
  const int I = B.I, O = B.O, nb = I / MX4_BLOCK;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
  const int o0 = blockIdx.x * 16, row0 = blockIdx.y * 16;
  // rows and outputs past the end repeat the last one; their sums are not stored
  const int o = min(o0 + n, O - 1), row = min(row0 + n, B.rows - 1);
  const uint8_t* wc = P.wc + (int64_t)o * (I / 2);
  const uint8_t* ws = P.ws + (int64_t)o * nb;
  const T* x = A4 ? nullptr : static_cast<const T*>(P.x) + (int64_t)row * I;
  const uint8_t* xc = A4 ? P.xc + (int64_t)row * (I / 2) : nullptr;
  const uint8_t* xs = A4 ? P.xs + (int64_t)row * nb : nullptr;

  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const u32x4 zero = {0u, 0u, 0u, 0u};
  for (int b = 4 * wave; b < nb; b += 4 * nw) {
    const bool ok = WHOLE || b + q < nb;
    const u32x4 w = ok ? *reinterpret_cast<const u32x4*>(wc + 16 * (b + q)) : zero;
    const uint32_t ex = mx4_exps<WHOLE>(ws, b, nb);
    const uint32_t e = (ex >> (8 * q)) & 255u;
    if constexpr (A4) {
      const u32x4 a = ok ? *reinterpret_cast<const u32x4*>(xc + 16 * (b + q)) : zero;
      const uint32_t ea = (mx4_exps<WHOLE>(xs, b, nb) >> (8 * q)) & 255u;
      acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(a), mx4_operand(w), acc, 4, 4, 0, (int)ea, 0,
                                                             (int)e);
    } else {
      u32x4 a[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) a[j] = ok ? *reinterpret_cast<const u32x4*>(x + 32 * (b + q) + 8 * j) : zero;
      const uint32_t emax = F16 ? max4(ex) : 0u;
      const float s = F16 ? mx4_relative(e, emax) : mx4_scale(e);
      f32x4 c = F16 ? (f32x4){0.f, 0.f, 0.f, 0.f} : acc;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        V wv;
        mx4_decode8(w[j], s, wv);
        c = mfma16x16x32(__builtin_bit_cast(V, a[j]), wv, c);
      }
      acc = F16 ? acc + mx4_factor(emax) * c : c;
    }
  }

  // lane: output n, rows 4 q .. +3
  __shared__ float part[16][16][17];
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][4 * q + i][n] = acc[i];
  __syncthreads();
  for (int t = tid; t < 256; t += blockDim.x) {
    const int r = t >> 4, c = t & 15;
    if (row0 + r >= B.rows || o0 + c >= O) continue;
    float v = part[0][r][c];
    for (int w = 1; w < nw; ++w) v += part[w][r][c];
    mx4_store<T>(P, row0 + r, o0 + c, O, v);
  }
}

template <typename T, bool A4>
static int mx4_rows_run(const Mx4Batch& b, int nprob, void* stream) {
  const int steps = (b.I + 127) / 128;
  const int nw = steps >= 64 ? 16 : steps >= 16 ? 8 : 4;
  const dim3 grid((unsigned)((b.O + 15) / 16), (unsigned)((b.rows + 15) / 16), (unsigned)nprob);
  if (b.I % 128 == 0)
    hipLaunchKernelGGL((mx4_rows_kernel<T, A4, true>), grid, dim3(64 * nw), 0, as_stream(stream), b);
  else
    hipLaunchKernelGGL((mx4_rows_kernel<T, A4, false>), grid, dim3(64 * nw), 0, as_stream(stream), b);
  return check_launch("mx4_rows_kernel");
}

// bytes of one quantised input, each part on a 256-byte boundary
static int64_t mx4_codes_bytes(int64_t rows, int64_t I) { return (rows * (I / 2) + 255) & ~(int64_t)255; }
static int64_t mx4_scales_bytes(int64_t rows, int64_t I) { return (rows * (I / MX4_BLOCK) + 255) & ~(int64_t)255; }

// Rows from which a product pays for materialising the weight.
static bool mx4_prefill(int64_t rows, int64_t I, int64_t O) { return rows > 256 && mx4h_supported(rows, I, O); }
// Quantised rows of more than one tile of the few-row kernel.
static bool mx4_gemm(int64_t rows, int64_t I, int64_t O) { return rows > 16 && mx4_gemm_supported(rows, O, I); }

}  // namespace rwkv7mi

using namespace rwkv7mi;

extern "C" int64_t rwkv7mi_mxfp4_linear_workspace_bytes(int nprob, int64_t rows, int64_t O, int64_t I, int act_dtype,
                                                        int quantize_input) {
  if (nprob < 1 || nprob > MX4_MAXPROB || rows <= 0 || O <= 0 || I <= 0) return 0;
  if (quantize_input && mx4_gemm(rows, I, O)) return mx4_gemm_workspace_bytes(nprob, rows, O, I);
  if (quantize_input) return nprob * (mx4_codes_bytes(rows, I) + mx4_scales_bytes(rows, I));
  return mx4_prefill(rows, I, O) ? mx4h_workspace_bytes(nprob, rows, I, O) : 0;
}

extern "C" int rwkv7mi_mxfp4_linear(int nprob, const void* const* x, const uint8_t* const* codes,
                                    const uint8_t* const* scales, const void* const* bias, const void* const* residual,
                                    void* const* y, const int* epilogue, int64_t rows, int64_t O, int64_t I,
                                    int act_dtype, int quantize_input, void* ws, int64_t ws_bytes, void* stream) {
  const std::string w("mxfp4_linear");
  if (!x || !codes || !scales || !y || !epilogue) return fail(RWKV7MI_EINVAL, w + ": null array");
  if (nprob < 1 || nprob > MX4_MAXPROB) return fail(RWKV7MI_EINVAL, w + ": 1..4 problems per launch");
  if (rows < 0 || O <= 0 || I <= 0) return fail(RWKV7MI_EINVAL, w + ": bad shape");
  if (I % MX4_BLOCK) return fail(RWKV7MI_EINVAL, w + ": in_features must be a multiple of 32");
  if (act_dtype != RWKV7MI_F16 && act_dtype != RWKV7MI_BF16)
    return fail(RWKV7MI_EINVAL, w + ": fp16 or bf16 activations");
  // (the row tiles are a grid dimension of at most 65535)
  if (rows > 16 * 65535 || O > INT32_MAX / 2 || I > INT32_MAX / 4) return fail(RWKV7MI_EINVAL, w + ": too large");
  if (rows == 0) return RWKV7MI_OK;
  Mx4Batch b{};
  b.rows = (int)rows;
  b.O = (int)O;
  b.I = (int)I;
  for (int i = 0; i < nprob; ++i) {
    Mx4Prob& p = b.p[i];
    p = Mx4Prob{x[i], nullptr, nullptr, codes[i], scales[i], bias ? bias[i] : nullptr,
                residual ? residual[i] : nullptr, y[i], epilogue[i]};
    if (!p.x || !p.wc || !p.ws || !p.y) return fail(RWKV7MI_EINVAL, w + ": null pointer");
    if ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.wc)) & 15)
      return fail(RWKV7MI_EINVAL, w + ": x and the codes must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(p.ws) & 3) return fail(RWKV7MI_EINVAL, w + ": the scales must be 4-byte aligned");
    if (p.epilogue < 0 || p.epilogue > 2) return fail(RWKV7MI_EINVAL, w + ": bad epilogue");
    if (p.epilogue == RWKV7MI_EPI_RESIDUAL && !p.residual) return fail(RWKV7MI_EINVAL, w + ": residual missing");
  }
  const bool bf = act_dtype == RWKV7MI_BF16;
  const int64_t need = rwkv7mi_mxfp4_linear_workspace_bytes(nprob, rows, O, I, act_dtype, quantize_input);
  if (need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < need))
    return fail(RWKV7MI_ESIZE, w + ": workspace missing, unaligned or smaller than "
                                   "rwkv7mi_mxfp4_linear_workspace_bytes");
  if (!quantize_input && mx4_prefill(rows, I, O)) return mx4h_run(b, nprob, act_dtype, ws, ws_bytes, stream);
  if (!quantize_input)
    return bf ? mx4_rows_run<__hip_bfloat16, false>(b, nprob, stream) : mx4_rows_run<__half, false>(b, nprob, stream);
  if (mx4_gemm(rows, I, O)) return mx4_gemm_run(b, nprob, act_dtype, ws, stream);
  uint8_t *xc[MX4_MAXPROB], *xs[MX4_MAXPROB];
  uint8_t* at = static_cast<uint8_t*>(ws);
  for (int i = 0; i < nprob; ++i) {
    b.p[i].xc = xc[i] = at;
    b.p[i].xs = xs[i] = at + mx4_codes_bytes(rows, I);
    at = xs[i] + mx4_scales_bytes(rows, I);
  }
  if (int rc = mx4_quantize_run(nprob, x, rows, I, I, act_dtype, xc, xs, stream)) return rc;
  return bf ? mx4_rows_run<__hip_bfloat16, true>(b, nprob, stream) : mx4_rows_run<__half, true>(b, nprob, stream);
}
