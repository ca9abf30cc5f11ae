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

// v (+ bias) through the epilogue, rounded once
template <typename T>
__device__ __forceinline__ void mx4_store(const Mx4Prob& P, int64_t row, int o, int O, float v) {
  const int64_t i = row * O + o;
  if (P.bias) v += ld(static_cast<const T*>(P.bias), o);
  if (P.epilogue == RWKV7MI_EPI_RELU2) {
    v = v > 0.f ? v : (v != v ? v : 0.f);  // (NaN stays)
    v = v * v;
  } else if (P.epilogue == RWKV7MI_EPI_RESIDUAL) {
    v += ld(static_cast<const T*>(P.residual), i);
  }
  static_cast<T*>(P.y)[i] = from_f32<T>(v);
}

// Quantises nprob inputs of [rows, I] values (row stride ld) into codes / scales (mx4.hip).
int mx4_quantize_run(int nprob, const void* const* x, int64_t rows, int64_t I, int64_t ld, int dtype,
                     uint8_t* const* codes, uint8_t* const* scales, void* stream);

}  // namespace rwkv7mi
