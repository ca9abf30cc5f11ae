// MXFP4 quantisation and its inverse.
//
// Per block of 32 inputs: e = clamp(floor(log2 amax) - 2 + 127, 0, 254), which
// puts the block's largest value at 4 <= |v| / 2^(e - 127) < 8, and each code is
// v / 2^(e - 127) rounded to nearest (ties to even), stopping at 6.  A block that
// holds an infinity or a NaN gets the scale NaN (255), so it shows in every
// product; its codes are 0.
//
// A lane takes 8 values; a block is four neighbouring lanes, whose maximum is
// two quad exchanges away.  Memory-bound: 2 (4) bytes a value in, 17/32 out: 16384 x 4096
// fp16 quantised and dequantised in 61 us, 5.5 TB/s with the codes that pass between.
#include "mx4_common.h"

namespace rwkv7mi {

namespace {

struct Mx4Quant {
  const void* x[MX4_MAXPROB];
  uint8_t *codes[MX4_MAXPROB], *scales[MX4_MAXPROB];
  int64_t rows, n8, ld;  // rows, runs of 8 values in all, row stride of x
  int row8;        // runs of 8 values in a row
  int in8;         // of which hold values (PADDED: the rest are zeros)
  // PADDED: the weights' scales too, in the workgroups from qblocks on
  const uint8_t* win[MX4_MAXPROB];
  uint32_t* wout[MX4_MAXPROB];
  int qblocks, O, nb, NS;
};

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));  // lane ^ 1
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));  // lane ^ 2
}

}  // namespace

// W's scales [O, nb] in the products' order [superstep][column][16], padded to whole
// supersteps (1.0 there): one thread a dword (the four blocks of lane half u in a step)
__device__ __forceinline__ void mx4_weight_scales(const Mx4Quant& Q, int p, int64_t t) {
  if (t >= (int64_t)Q.O * 4 * Q.NS) return;
  const int o = (int)(t / (4 * Q.NS)), d = (int)(t % (4 * Q.NS)), b0 = 16 * (d >> 2) + 8 * (d & 1) + (d >> 1 & 1);
  const uint8_t* s = Q.win[p] + (int64_t)o * Q.nb;
  uint32_t v = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = b0 + 2 * i;
    v |= (b < Q.nb ? (uint32_t)s[b] : 127u) << (8 * i);
  }
  Q.wout[p][((int64_t)(d >> 2) * Q.O + o) * 4 + (d & 3)] = v;
}

// PADDED: rows padded to whole supersteps, their scales in the GEMM's order; the
// same launch orders the weights' scales (a launch of their own took 4 us)
template <typename T, bool PADDED>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const Mx4Quant Q) {
  const int p = blockIdx.y;
  if (PADDED && (int)blockIdx.x >= Q.qblocks) {
    mx4_weight_scales(Q, p, (int64_t)(blockIdx.x - Q.qblocks) * 256 + threadIdx.x);
    return;
  }
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= Q.n8) return;  // (n8 is a multiple of 4: a block's lanes stay together)
  const int64_t row = t / Q.row8;
  const int run = (int)(t - row * Q.row8);
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (!PADDED || run < Q.in8) ld8(static_cast<const T*>(Q.x[p]) + row * Q.ld + 8 * (int64_t)run, v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  m = quad_max(m);
  const int ex = (int)(m >> 23);  // floor(log2 amax) + 127 (0 below the normal range)
  const uint32_t e = ex == 255 ? 255u : (uint32_t)max(ex - 2, 0);
  uint32_t d = 0;
  if (ex != 255) {
    const float s = mx4_scale(e);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[0], v[1], s, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[2], v[3], s, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[4], v[5], s, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, v[6], v[7], s, 3);
  }
  reinterpret_cast<uint32_t*>(Q.codes[p])[t] = d;
  if ((t & 3) == 0) {
    int64_t b = t >> 2;
    if (PADDED)  // [superstep][row][16]
      b = ((run >> 6) * Q.rows + row) * 16 + ((b & 1) << 3 | (b >> 3 & 1) << 2 | (b >> 1 & 3));
    Q.scales[p][b] = (uint8_t)e;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ scales, T* __restrict__ y,
                                                             int64_t n8) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= n8) return;
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const uint32_t d = codes[t];
  const float s = mx4_scale(scales[t >> 2]);
  const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 1);
  const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d, s, 3);
  const float v[8] = {a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
  st8(y + 8 * t, v);
}

static int mx4_quantize_go(Mx4Quant& q, int nprob, const void* const* x, int64_t rows, int64_t I, int64_t ld, int dtype,
                           bool padded, uint8_t* const* codes, uint8_t* const* scales, void* stream) {
  for (int i = 0; i < nprob; ++i) {
    q.x[i] = x[i];
    q.codes[i] = codes[i];
    q.scales[i] = scales[i];
  }
  q.rows = rows;
  q.in8 = (int)(I / 8);
  q.row8 = padded ? q.NS * 64 : q.in8;
  q.n8 = rows * q.row8;
  q.ld = ld;
  q.qblocks = (int)((q.n8 + 255) / 256);
  const dim3 grid((unsigned)(q.qblocks + (padded ? ((int64_t)q.O * 4 * q.NS + 255) / 256 : 0)), (unsigned)nprob);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (padded)
      hipLaunchKernelGGL((mx4_quantize_kernel<T, true>), grid, dim3(256), 0, as_stream(stream), q);
    else
      hipLaunchKernelGGL((mx4_quantize_kernel<T, false>), grid, dim3(256), 0, as_stream(stream), q);
    return check_launch("mx4_quantize_kernel");
  });
}
int mx4_quantize_run(int nprob, const void* const* x, int64_t rows, int64_t I, int64_t ld, int dtype,
                     uint8_t* const* codes, uint8_t* const* scales, void* stream) {
  Mx4Quant q{};
  return mx4_quantize_go(q, nprob, x, rows, I, ld, dtype, false, codes, scales, stream);
}
int mx4_quantize_padded(const Mx4Batch& b, int nprob, int dtype, uint8_t* const* codes, uint8_t* const* scales,
                        uint8_t* const* wscales, void* stream) {
  Mx4Quant q{};
  const void* x[MX4_MAXPROB];
  for (int i = 0; i < nprob; ++i) {
    x[i] = b.p[i].x;
    q.win[i] = b.p[i].ws;
    q.wout[i] = reinterpret_cast<uint32_t*>(wscales[i]);
  }
  q.O = b.O;
  q.nb = b.I / MX4_BLOCK;
  q.NS = (b.I + 511) / 512;
  return mx4_quantize_go(q, nprob, x, b.rows, b.I, b.I, dtype, true, codes, scales, stream);
}

}  // namespace rwkv7mi

using namespace rwkv7mi;

// shapes both entries take: whole blocks, a grid the launch can hold
static int mx4_shape(const char* who, int64_t rows, int64_t I) {
  const std::string w(who);
  if (rows < 0 || I <= 0) return fail(RWKV7MI_EINVAL, w + ": bad shape");
  if (I % MX4_BLOCK) return fail(RWKV7MI_EINVAL, w + ": the row length must be a multiple of 32");
  // (a launch holds fewer than 2^32 lanes of 8 values)
  if (I > INT32_MAX || rows > (((int64_t)1 << 35) - 2048) / I) return fail(RWKV7MI_EINVAL, w + ": too large");
  return RWKV7MI_OK;
}

extern "C" int rwkv7mi_mxfp4_quantize(const void* x, int64_t rows, int64_t I, int64_t ld, int dtype, uint8_t* codes,
                                      uint8_t* scales, void* stream) {
  if (int rc = mx4_shape("mxfp4_quantize", rows, I)) return rc;
  if (!valid_dtype(dtype)) return fail(RWKV7MI_EINVAL, "mxfp4_quantize: bad dtype");
  if (ld < I) return fail(RWKV7MI_EINVAL, "mxfp4_quantize: bad row stride");
  if (rows == 0) return RWKV7MI_OK;
  if (!x || !codes || !scales) return fail(RWKV7MI_EINVAL, "mxfp4_quantize: null pointer");
  const int64_t es = dtype == RWKV7MI_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) & 15) || (ld * es) % 16 || (reinterpret_cast<uintptr_t>(codes) & 3))
    return fail(RWKV7MI_EINVAL, "mxfp4_quantize: rows must start 16-byte aligned, codes 4-byte aligned");
  return mx4_quantize_run(1, &x, rows, I, ld, dtype, &codes, &scales, stream);
}

extern "C" int rwkv7mi_mxfp4_dequantize(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t I, void* y,
                                        int dtype, void* stream) {
  if (int rc = mx4_shape("mxfp4_dequantize", rows, I)) return rc;
  if (!valid_dtype(dtype)) return fail(RWKV7MI_EINVAL, "mxfp4_dequantize: bad dtype");
  if (rows == 0) return RWKV7MI_OK;
  if (!codes || !scales || !y) return fail(RWKV7MI_EINVAL, "mxfp4_dequantize: null pointer");
  if ((reinterpret_cast<uintptr_t>(y) & 15) || (reinterpret_cast<uintptr_t>(codes) & 3))
    return fail(RWKV7MI_EINVAL, "mxfp4_dequantize: y must be 16-byte aligned, codes 4-byte aligned");
  const int64_t n8 = rows * (I / 8);
  return dispatch_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(mx4_dequantize_kernel<T>, dim3((unsigned)((n8 + 255) / 256)), dim3(256), 0, as_stream(stream),
                       reinterpret_cast<const uint32_t*>(codes), scales, static_cast<T*>(y), n8);
    return check_launch("mx4_dequantize_kernel");
  });
}
