// MXFP4 helpers shared by the quantiser (mx4.hip) and the products
// (mx4_linear.hip).
//
// Format (the OCP microscaling MXFP4): 32 consecutive inputs of a row share one
// power-of-two scale byte e, 2^(e - 127) (255: NaN), and a 4-bit e2m1 code each:
// 0, 0.5, 1, 1.5, 2, 3, 4, 6 and the sign in bit 3.  codes [rows, I/2] hold the
// even input in the low nibble, scales [rows, I/32].
#pragma once
#include <type_traits>

#include "common.h"

namespace rwkv7mi {

constexpr int MX4_BLOCK = 32;
constexpr int MX4_MAXPROB = 4;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// One product y = epilogue(x W^T + bias) of a launch.
struct Mx4Prob {
  const void* x;          // 16-bit rows [rows, I]
  const uint8_t *xc, *xs; // or their MXFP4 form
  const uint8_t *wc, *ws; // codes [O, I/2], scales [O, I/32]
  const void *bias, *residual;
  void* y;
  int epilogue;
};
struct Mx4Batch {
  Mx4Prob p[MX4_MAXPROB];
  int rows, O, I;
};

// The float 2^(e - 127) as the conversions take it (they use the exponent
// field alone; 255 gives NaN).
__device__ __forceinline__ float mx4_scale(uint32_t e) { return __uint_as_float(e << 23); }

// 16-bit weights are formed over a run of inputs whose largest scale byte is emax, their
// codes times 2^(byte - 127), and the sums over the run take a factor in fp32 (NaN for
// emax = 255).
//  * fp16: scaled relative to emax, 2^(13 + e - emax) (at most 6 x 2^13, exact down to
//    2^-36 of the largest scale, rounding at 2^-24 below).
//  * bf16 holds a code times 2^(e - 127) exactly for e up to 252; 6 x 2^126 is past its
//    range (and fp32's).  Runs with a byte of 253 or 254 are formed at a quarter (their
//    bytes 0 and 1, 2^-251 of the largest at most, at no less than 2^-127).
template <typename T>
__device__ __forceinline__ uint32_t mx4_run_byte(uint32_t e, uint32_t emax) {
  if constexpr (std::is_same<T, __half>::value)
    return (uint32_t)max(140 + (int)e - (int)emax, 1);
  else
    return emax < 253u ? e : (uint32_t)max((int)e - 2, 0);
}
template <typename T>
__device__ __forceinline__ float mx4_run_factor(uint32_t emax) {
  if (emax == 255u) return __builtin_nanf("");
  if constexpr (std::is_same<T, __half>::value)
    return ldexpf(1.f, (int)emax - 140);
  else
    return emax < 253u ? 1.f : 4.f;
}
// an emax of that factor
template <typename T>
__device__ __forceinline__ uint32_t mx4_factor_emax(float f) {
  if constexpr (std::is_same<T, __half>::value)
    return f != f ? 255u : (uint32_t)(ilogbf(f) + 140);
  else
    return f == 1.f ? 0u : 254u;
}

__device__ __forceinline__ uint32_t mx4_max4(uint32_t v) {  // the largest byte
  return max(max(v & 255u, (v >> 8) & 255u), max((v >> 16) & 255u, v >> 24));
}

// 8 codes of a dword -> 8 values times the scale, in order
__device__ __forceinline__ void mx4_decode8(uint32_t d, float s, bf16x8& o) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 0);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 1);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 2);
  const bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(d, s, 3);
  o = (bf16x8){a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}
__device__ __forceinline__ void mx4_decode8(uint32_t d, float s, f16x8& o) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 0);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 1);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 2);
  const f16x2 e = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(d, s, 3);
  o = (f16x8){a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

template <typename T> struct Mx4Types { typedef f16x8 V; };
template <> struct Mx4Types<__hip_bfloat16> { typedef bf16x8 V; };

__device__ __forceinline__ float mx4_relu2(float v) {
  v = v < 0.f ? 0.f : v;  // (NaN stays)
  return v * v;
}

// v (+ bias) through the epilogue, rounded once
template <typename T>
__device__ __forceinline__ void mx4_store(const Mx4Prob& P, int64_t row, int o, int O, float v) {
  const int64_t i = row * O + o;
  if (P.bias) v += ld(static_cast<const T*>(P.bias), o);
  if (P.epilogue == RWKV7MI_EPI_RELU2) {
    v = mx4_relu2(v);
  } else if (P.epilogue == RWKV7MI_EPI_RESIDUAL) {
    v += ld(static_cast<const T*>(P.residual), i);
  }
  static_cast<T*>(P.y)[i] = from_f32<T>(v);
}

// Quantises nprob inputs of [rows, I] values (row stride ld) into codes / scales (mx4.hip).
int mx4_quantize_run(int nprob, const void* const* x, int64_t rows, int64_t I, int64_t ld, int dtype,
                     uint8_t* const* codes, uint8_t* const* scales, void* stream);
// The same for the products of b, rows padded with zeros to NS = ceil(I / 512) supersteps: codes [rows, 256 NS]
// bytes, scales [NS, rows, 16] with block 8 s + 2 h + u of a superstep at byte 8 u + 4 s + h, and the weights'
// scales in that order, wscales [NS, O, 16].
int mx4_quantize_padded(const Mx4Batch& b, int nprob, int dtype, uint8_t* const* codes, uint8_t* const* scales,
                        uint8_t* const* wscales, void* stream);

// Products of two MXFP4 operands of many rows (mx4_gemm.hip): x is quantised there.
bool mx4_gemm_supported(int64_t rows, int64_t O, int64_t I);
int64_t mx4_gemm_workspace_bytes(int nprob, int64_t rows, int64_t O, int64_t I);
int mx4_gemm_run(const Mx4Batch& b, int nprob, int act_dtype, void* ws, void* stream);

// Products with 16-bit rows, many of them (mx4_tile.hip).
bool mx4_tile_supported(int64_t rows, int64_t O, int64_t I);
int64_t mx4_tile_workspace_bytes(int nprob, int64_t rows, int64_t O, int64_t I);
double mx4_tile_us(int nprob, int64_t rows, int64_t O, int64_t I);  // an estimate
int mx4_tile_run(const Mx4Batch& b, int nprob, int act_dtype, void* ws, void* stream);

// Products through fp16 / bf16 records of the weight and the 256 x 256 GEMM of
// mm8h.hip: whether it takes these shapes, its workspace, its launches.
bool mx4h_supported(int64_t rows, int64_t I, int64_t O);
int64_t mx4h_workspace_bytes(int nprob, int64_t I, int64_t O);
int mx4h_run(const Mx4Batch& b, int nprob, int act_dtype, void* ws, int64_t ws_bytes, void* stream);

}  // namespace rwkv7mi
