// Products with an MXFP4 weight: y = epilogue(x W^T + bias), fp16 / bf16 rows
// x, or the same rows quantised to MXFP4 on the way.
//
// mx4_rows_kernel, 16 rows a tile, few of them: the nw waves of a workgroup share K in units of
// 512 inputs and go through groups of 16 outputs, a grid apart; a group's fp32 sums
// meet in LDS in wave order.  A unit is four steps of 128 inputs (four blocks): lane
// n + 16 q holds block q of output n, 16 bytes of codes and one scale byte, which is
// the operand of
//  * one v_mfma_scale_f32_16x16x128_f8f6f4 where x is MXFP4 too, or
//  * four v_mfma_f32_16x16x32 where x is 16-bit: MFMA j takes inputs 8 j .. +7
//    of every lane's block, and so do the rows of x.
// A wave has one unit: its part of x stays in registers for all its groups (32 rows of
// it from 17 rows on, whose codes are then converted once: 64 x 4096 -> 4096 16.1 ->
// 14.6 us), and the next group's codes and scales are loaded before this one's MFMAs.
// Above the 16 units (8 with 32 rows) that a CU's registers hold the units go over
// several workgroups, and a second launch adds their sums (16 x 16384 -> 4096 with two
// units a wave, x reloaded, 25.6 us).  What does not carry weights is kept out of the
// loads' way: a group's scales are loaded once by the workgroup, through LDS, a group
// ahead (by each wave 1.4 us more at 1 x 4096 -> 16384, 13.1 us then), and 16-bit rows
// by whole lines, through LDS (in the operand's layout, 16 bytes of 64 lines an
// instruction, 17.3 us for 14.6 at 16 x 4096 -> 16384).  Neither 16-bit type holds a code
// times every scale, so the codes of a step (bf16: of a unit) are scaled by its largest
// scale and the sums by that one's factor (mx4_common.h).
//
// 8 x 4096 -> 65536 takes 33.5 us, 4.3 TB/s of the 5.4 that a copy reaches.  Smaller
// weights are bound by latency, a chain of x, the first codes and the sums' meeting in
// LDS: 1 x 4096 -> 16384 11.8 us for the 6.6 of its bytes (9.5 with them in the caches),
// 16 x 4096 -> 16384 14.6 to 15.0; with the second launch 1 x 16384 -> 4096 14.3, 16 rows
// 17.7 (the same bytes).
#include <algorithm>

#include "mx4_common.h"

namespace rwkv7mi {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 mx4_operand(u32x4 v) {
  return (i32x8){(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}

// The scale bytes of a row's unit (16 blocks from b), a dword a step, block q of it
// in byte q; blocks past the row read 0.  SC: 2 where I % 512 == 0 (16 aligned
// bytes), 1 where I % 128 == 0 (aligned dwords), else bytes.
template <int SC>
__device__ __forceinline__ u32x4 mx4_unit_scales(const uint8_t* row, int b, int nb) {
  if constexpr (SC == 2) return *reinterpret_cast<const u32x4*>(row + b);
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    if constexpr (SC == 1) {
      if (b + 4 * s < nb) v[s] = *reinterpret_cast<const uint32_t*>(row + b + 4 * s);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (b + 4 * s + i < nb) v[s] |= (uint32_t)row[b + 4 * s + i] << (8 * i);
    }
  }
  return v;
}

}  // namespace

struct Mx4Rows {
  Mx4Batch b;
  int S;        // workgroups that share K
  float* part;  // S > 1: [problem][split][row][O]
};

// RT: 16-row tiles a wave
template <typename T, bool A4, int SC, int RT>
__global__ __launch_bounds__(RT > 1 ? 512 : 1024) void mx4_rows_kernel(const Mx4Rows R) {
  using V = typename Mx4Types<T>::V;
  constexpr bool F16 = std::is_same<T, __half>::value && !A4;
  const Mx4Batch& B = R.b;
  const Mx4Prob& P = B.p[blockIdx.z / R.S];
  const int I = B.I, O = B.O, nb = I / MX4_BLOCK, groups = (O + 15) / 16;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), nw = blockDim.x >> 6;
  const int row0 = blockIdx.y * 16 * RT;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  constexpr int NX = A4 ? 1 : 4;  // 16-byte pieces of x a step

  // [group's parity][output][wave] scales, then [group's parity][wave][row][output]
  // sums in the memory that first holds [wave][row][16-byte piece] of a step of x
  extern __shared__ __align__(16) char smem[];
  u32x4* const scale = reinterpret_cast<u32x4*>(smem);
  char* const lower = smem + 512 * nw;
  typedef float Sums[16 * RT][17];
  Sums* const part = reinterpret_cast<Sums*>(lower);
  u32x4* const xl = reinterpret_cast<u32x4*>(lower) + wave * 256;

  u32x4 w[4], wn[4], a[RT][4][NX], ea = zero;
  const int u0 = (int)(blockIdx.z % R.S) * nw;
  const int b0 = 16 * (u0 + wave);  // (waves past the last unit add zeros)
  const bool has = b0 < nb;
  auto load_w = [&](int g, u32x4 (&w)[4]) {
    const int64_t o = min(16 * g + n, O - 1);  // (outputs past the end repeat the last one and are not stored)
    const uint8_t* wc = P.wc + o * (I / 2) + 16 * (b0 + q);
#pragma unroll
    for (int s = 0; s < 4; ++s)
      w[s] = SC == 2 || b0 + 4 * s + q < nb ? *reinterpret_cast<const u32x4*>(wc + 64 * s) : zero;
  };
  // thread t: the scales of output t / nw, unit t % nw of the group
  const int so = tid / nw, su = tid % nw, sb = 16 * (u0 + su);
  const bool scales = tid < 16 * nw && sb < nb;
  auto load_s = [&](int g) {
    return mx4_unit_scales<SC>(P.ws + (int64_t)min(16 * g + so, O - 1) * nb, sb, nb);
  };
  u32x4 sn = zero;
  if (has) load_w(blockIdx.x, w);
  if (scales) scale[so * nw + su] = load_s(blockIdx.x);
  if (has) {
    if constexpr (A4) {
      const bool mine = row0 + n < B.rows;
      const int64_t row = min(row0 + n, B.rows - 1);
#pragma unroll
      for (int s = 0; s < 4; ++s)
        a[0][s][0] = mine && (SC == 2 || b0 + 4 * s + q < nb)
                         ? *reinterpret_cast<const u32x4*>(P.xc + row * (I / 2) + 16 * (b0 + 4 * s + q)) : zero;
      ea = mine ? mx4_unit_scales<SC>(P.xs + row * nb, b0, nb) : zero;
    } else {
      // load v of a step: lane, piece lane % 16 of row 4 v + lane / 16.  (Rows past the end
      // hold anything and are not stored.)
      const T* x = static_cast<const T*>(P.x) + 32 * b0 + 8 * n;
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const int r = row0 + 16 * t + 4 * v + q;
#pragma unroll
          for (int s = 0; s < 4; ++s) a[t][s][v] = zero;
          if (r < B.rows) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
              if (SC == 2 || 32 * b0 + 128 * s + 8 * n < I)
                a[t][s][v] = *reinterpret_cast<const u32x4*>(x + (int64_t)r * I + 128 * s);
          }
        }
      // piece p of row r at p ^ r: rows of 256 bytes without bank conflicts either way
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
          for (int v = 0; v < 4; ++v)
            if (row0 + 16 * t + 4 * v < B.rows) xl[16 * (4 * v + q) + (n ^ (4 * v + q))] = a[t][s][v];
#pragma unroll
          for (int j = 0; j < 4; ++j) a[t][s][j] = xl[16 * n + ((4 * q + j) ^ n)];
        }
    }
  }
  __syncthreads();
  int par = 0;
  for (int g = blockIdx.x; g < groups; g += gridDim.x, par ^= 1) {
    f32x4 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const bool next = g + (int)gridDim.x < groups;
    if (next && scales) sn = load_s(g + gridDim.x);
    if (has) {
      if (next) load_w(g + gridDim.x, wn);
      const u32x4 e = scale[(16 * par + n) * nw + wave];
      // bf16: the unit is the run
      const uint32_t unit = A4 || F16 ? 0u : max(max(mx4_max4(e[0]), mx4_max4(e[1])), max(mx4_max4(e[2]), mx4_max4(e[3])));
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const uint32_t ew = e[s], eb = (ew >> (8 * q)) & 255u;
        if constexpr (A4) {
          acc[0] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(a[0][s][0]), mx4_operand(w[s]), acc[0], 4, 4,
                                                                    0, (int)((ea[s] >> (8 * q)) & 255u), 0, (int)eb);
        } else {
          const uint32_t emax = F16 ? mx4_max4(ew) : unit;
          const float sc = mx4_scale(mx4_run_byte<T>(eb, emax));
          f32x4 c[RT];
#pragma unroll
          for (int t = 0; t < RT; ++t) c[t] = F16 ? (f32x4){0.f, 0.f, 0.f, 0.f} : acc[t];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            V wv;
            mx4_decode8(w[s][j], sc, wv);
#pragma unroll
            for (int t = 0; t < RT; ++t) c[t] = mfma16x16x32(__builtin_bit_cast(V, a[t][s][j]), wv, c[t]);
          }
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t] = F16 ? acc[t] + mx4_run_factor<T>(emax) * c[t] : c[t];
        }
      }
      if constexpr (!A4 && !F16) {
#pragma unroll
        for (int t = 0; t < RT; ++t) acc[t] = acc[t] * mx4_run_factor<T>(unit);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) w[s] = wn[s];
    }
    if (next && scales) scale[(16 * (par ^ 1) + so) * nw + su] = sn;
    // lane: output n, rows 4 q .. +3 of each tile.  (A wave is at most one group ahead of the
    // readers of the other half.)
#pragma unroll
    for (int i = 0; i < 4 * RT; ++i) part[par * nw + wave][16 * (i >> 2) + 4 * q + (i & 3)][n] = acc[i >> 2][i & 3];
    __syncthreads();
    for (int z = tid; z < 256 * RT; z += blockDim.x) {
      const int r = z >> 4, c = z & 15;
      if (row0 + r >= B.rows || 16 * g + c >= O) continue;
      float v = part[par * nw][r][c];
      for (int k = 1; k < nw; ++k) v += part[par * nw + k][r][c];
      if (R.S > 1)
        R.part[((int64_t)blockIdx.z * B.rows + row0 + r) * O + 16 * g + c] = v;
      else
        mx4_store<T>(P, row0 + r, 16 * g + c, O, v);
    }
  }
}

// One thread an output: its S partial sums in split order
template <typename T>
__global__ __launch_bounds__(256) void mx4_rows_reduce_kernel(const Mx4Rows R) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x, each = (int64_t)R.b.rows * R.b.O;
  if (t >= each) return;
  const float* p = R.part + blockIdx.y * R.S * each + t;
  float v = p[0];
  for (int z = 1; z < R.S; ++z) v += p[z * each];
  mx4_store<T>(R.b.p[blockIdx.y], t / R.b.O, (int)(t % R.b.O), R.b.O, v);
}

// Workgroups that share K: up to 16 units of 512 inputs in one, 8 where there are
// more (16 x 16384 -> 4096: 0.8 us less with 8 than with 16, and for 1 row).
static int mx4_rows_tiles(int64_t rows, bool A4) { return rows <= 16 || A4 ? 1 : 2; }
static int mx4_rows_splits(int64_t rows, int64_t I, bool A4) {
  return I <= (mx4_rows_tiles(rows, A4) > 1 ? 4096 : 8192) ? 1 : (int)((I + 4095) / 4096);
}
static int64_t mx4_rows_part_bytes(int nprob, int64_t rows, int64_t O, int64_t I, bool A4) {
  const int S = mx4_rows_splits(rows, I, A4);
  return S > 1 ? nprob * S * rows * O * 4 : 0;
}

// LDS bytes a wave: its scales, and its sums or its part of x
static int mx4_rows_lds(int rt, bool A4) { return 512 + std::max(2 * 16 * rt * 17 * 4, A4 ? 0 : 4096); }

template <typename T, bool A4>
static int mx4_rows_run(const Mx4Batch& b, int nprob, void* part, void* stream) {
  Mx4Rows r{b, mx4_rows_splits(b.rows, b.I, A4), static_cast<float*>(part)};
  const int units = (b.I + 511) / 512, nw = (units + r.S - 1) / r.S, rt = mx4_rows_tiles(b.rows, A4);
  const int groups = (b.O + 15) / 16, tiles = (b.rows + 16 * rt - 1) / (16 * rt);
  // 16 waves a CU fit by registers (8 with two tiles of 16-bit rows): no more workgroups than run at once
  const int fit = rt > 1 ? 8 : 16;
  const int64_t most = std::max<int64_t>(1, 256 * (fit / nw) / ((int64_t)tiles * nprob * r.S));
  const dim3 grid((unsigned)std::min<int64_t>(groups, most), (unsigned)tiles, (unsigned)(nprob * r.S));
  // (16-byte scale reads need the rows of scales to start 16-byte aligned)
  bool wide = b.I % 512 == 0;
  for (int i = 0; i < nprob; ++i)
    if ((reinterpret_cast<uintptr_t>(b.p[i].ws) | reinterpret_cast<uintptr_t>(b.p[i].xs)) & 15) wide = false;
  const int lds = nw * mx4_rows_lds(rt, A4);
  const auto go = [&](auto sc) {
    constexpr int SC = decltype(sc)::value;
    static std::atomic<uint64_t> raised[2];
    const auto launch = [&](auto kern, std::atomic<uint64_t>& done) {
      if (lds > 65536)
        if (int rc = raise_dynamic_lds(reinterpret_cast<const void*>(kern), 16 * mx4_rows_lds(1, A4), done, "mx4_rows_kernel"))
          return rc;
      hipLaunchKernelGGL(kern, grid, dim3(64 * nw), lds, as_stream(stream), r);
      return check_launch("mx4_rows_kernel");
    };
    if constexpr (!A4)
      if (rt == 2) return launch(&mx4_rows_kernel<T, A4, SC, 2>, raised[1]);
    return launch(&mx4_rows_kernel<T, A4, SC, 1>, raised[0]);
  };
  if (int rc = wide               ? go(std::integral_constant<int, 2>{})
               : b.I % 128 == 0 ? go(std::integral_constant<int, 1>{})
                                : go(std::integral_constant<int, 0>{}))
    return rc;
  if (r.S == 1) return RWKV7MI_OK;
  const int64_t each = (int64_t)b.rows * b.O;
  hipLaunchKernelGGL(mx4_rows_reduce_kernel<T>, dim3((unsigned)((each + 255) / 256), (unsigned)nprob), dim3(256), 0,
                     as_stream(stream), r);
  return check_launch("mx4_rows_reduce_kernel");
}

// bytes of one quantised input, each part on a 256-byte boundary
static int64_t mx4_codes_bytes(int64_t rows, int64_t I) { return (rows * (I / 2) + 255) & ~(int64_t)255; }
static int64_t mx4_scales_bytes(int64_t rows, int64_t I) { return (rows * (I / MX4_BLOCK) + 255) & ~(int64_t)255; }

// A call of the few-row kernel with 17 to 512 16-bit rows, in us: a start and its
// workgroups' rounds of a group of outputs each, which take about the same time at any K
// (fitted to 24 shapes: 128 x 4096 -> 4096, 4 rounds, 16.5 and estimated 16.0, 384 rows,
// 13 rounds, 38.3 and 38.5; 320 x 1216 -> 8088, 10 rounds with ragged K, 43.2 and 43.0).
static double mx4_rows_us(int nprob, int64_t rows, int64_t O, int64_t I) {
  const int64_t S = mx4_rows_splits(rows, I, false), nw = ((I + 511) / 512 + S - 1) / S;
  const int64_t share = (rows + 31) / 32 * nprob * S, groups = (O + 15) / 16, fit = 256 * (8 / nw);
  const int64_t wide = std::min(groups, std::max<int64_t>(1, fit / share));
  const int64_t rounds = (groups + wide - 1) / wide * ((wide * share + fit - 1) / fit);
  return 6.0 + (I % 512 ? 3.7 : 2.5) * rounds + (S > 1 ? 3.0 : 0.0);
}

// Which kernel takes a product.  The few-row kernel: up to 16 rows, and up to 512 where
// its passes over the weight, one a tile of 32 rows, are estimated to take no longer than
// the larger tiles.  16-bit rows on it and on those: 128 x 4096 -> 4096 16.5 and 23.4 us,
// 40 x 8192 -> 2048 13.1 and 19.5, 256 x 4096 -> 4096 25.6 and 26.7, 32 x 4096 -> 65536
// 52.5 and 57.3; 96 x 4096 -> 16384 41.5 and 34.8, 128 x 16384 -> 4096 51.7 and 39.5.
// MXFP4 rows, 16 a tile, by rows x weight: 128 x 4096 -> 4096 16.6 and 19.7, 64 x 4096 ->
// 16384 26.0 and 26.0.  And what the others' offsets cannot hold.  Else the 64- to
// 256-row tiles.  16-bit rows from 1024
// tiles of 256 x 256 on write the weight out in 16 bits and run the GEMM of mm8h.hip:
// without conversions between its MFMAs it holds a higher clock over such long calls
// (16384 x 4096 -> 16384 1636 us, on the tiles 2000), and the pass over the weight
// is small against them (1000 rows, 256 tiles: 150 and 115).
enum Mx4Route { MX4_ROWS, MX4_TILE, MX4_GEMM, MX4_PREFILL };
static Mx4Route mx4_route(int nprob, int64_t rows, int64_t I, int64_t O, int quantize_input) {
  if (rows <= 16) return MX4_ROWS;
  if (quantize_input && rows <= 256 && (rows + 15) / 16 * (O * I) <= 1 << 27) return MX4_ROWS;
  if (quantize_input) return mx4_gemm_supported(rows, O, I) ? MX4_GEMM : MX4_ROWS;
  if ((rows + 255) / 256 * ((O + 255) / 256) >= 1024 && mx4h_supported(rows, I, O)) return MX4_PREFILL;
  if (!mx4_tile_supported(rows, O, I)) return MX4_ROWS;
  return rows <= 512 && mx4_rows_us(nprob, rows, O, I) <= mx4_tile_us(nprob, rows, O, I) ? MX4_ROWS : MX4_TILE;
}

// The quantiser's launch of a product's rows (mx4.hip: 8 values a lane; before the GEMM
// rows padded to whole supersteps, and the weight's scales) holds fewer than 2^32 lanes.
static bool mx4_quantizable(Mx4Route route, int64_t rows, int64_t I, int64_t O) {
  const int64_t NS = (I + 511) / 512;
  return (route == MX4_GEMM ? 64 * NS * rows + 4 * NS * O : rows * (I / 8)) <= ((int64_t)1 << 32) - 1024;
}

}  // namespace rwkv7mi

using namespace rwkv7mi;

extern "C" int64_t rwkv7mi_mxfp4_linear_workspace_bytes(int nprob, int64_t rows, int64_t O, int64_t I, int act_dtype,
                                                        int quantize_input) {
  if (nprob < 1 || nprob > MX4_MAXPROB || rows <= 0 || O <= 0 || I <= 0) return 0;
  const Mx4Route route = mx4_route(nprob, rows, I, O, quantize_input);
  if (quantize_input && !mx4_quantizable(route, rows, I, O)) return 0;
  if (route == MX4_PREFILL) return mx4h_workspace_bytes(nprob, I, O);
  if (route == MX4_GEMM) return mx4_gemm_workspace_bytes(nprob, rows, O, I);
  if (route == MX4_TILE) return mx4_tile_workspace_bytes(nprob, rows, O, I);
  const int64_t part = mx4_rows_part_bytes(nprob, rows, O, I, quantize_input);
  return part + (quantize_input ? nprob * (mx4_codes_bytes(rows, I) + mx4_scales_bytes(rows, I)) : 0);
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
  const Mx4Route route = mx4_route(nprob, rows, I, O, quantize_input);
  if (quantize_input && !mx4_quantizable(route, rows, I, O))
    return fail(RWKV7MI_EINVAL, w + ": too large to quantise (split the rows)");
  const int64_t need = rwkv7mi_mxfp4_linear_workspace_bytes(nprob, rows, O, I, act_dtype, quantize_input);
  if (need && (!ws || (reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < need))
    return fail(RWKV7MI_ESIZE, w + ": workspace missing, unaligned or smaller than "
                                   "rwkv7mi_mxfp4_linear_workspace_bytes");
  if (route == MX4_PREFILL) return mx4h_run(b, nprob, act_dtype, ws, ws_bytes, stream);
  if (route == MX4_GEMM) return mx4_gemm_run(b, nprob, act_dtype, ws, stream);
  if (route == MX4_TILE) return mx4_tile_run(b, nprob, act_dtype, ws, stream);
  if (!quantize_input)
    return bf ? mx4_rows_run<__hip_bfloat16, false>(b, nprob, ws, stream)
              : mx4_rows_run<__half, false>(b, nprob, ws, stream);
  uint8_t *xc[MX4_MAXPROB], *xs[MX4_MAXPROB];
  uint8_t* at = static_cast<uint8_t*>(ws);
  for (int i = 0; i < nprob; ++i) {
    b.p[i].xc = xc[i] = at;
    b.p[i].xs = xs[i] = at + mx4_codes_bytes(rows, I);
    at = xs[i] + mx4_scales_bytes(rows, I);
  }
  if (int rc = mx4_quantize_run(nprob, x, rows, I, I, act_dtype, xc, xs, stream)) return rc;
  return bf ? mx4_rows_run<__hip_bfloat16, true>(b, nprob, at, stream) : mx4_rows_run<__half, true>(b, nprob, at, stream);
}

extern "C" int rwkv7mi_mxfp4_linear1(const void* x, const uint8_t* codes, const uint8_t* scales, const void* bias,
                                     const void* residual, void* y, int epilogue, int64_t rows, int64_t O, int64_t I,
                                     int act_dtype, int quantize_input, void* ws, int64_t ws_bytes, void* stream) {
  return rwkv7mi_mxfp4_linear(1, &x, &codes, &scales, &bias, &residual, &y, &epilogue, rows, O, I, act_dtype,
                              quantize_input, ws, ws_bytes, stream);
}
