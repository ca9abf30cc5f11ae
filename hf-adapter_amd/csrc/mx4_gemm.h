// What the two many-row MXFP4 products share (mx4_gemm.hip: 4-bit rows, mx4_tile.hip:
// 16-bit rows): the 64 MI x 256 tile of a workgroup, two rows of WC waves of 32 MI x 256
// / WC in tiles of 32x32 MFMAs, W as the A operand, its numbering, its epilogue, the
// plan of tile heights and K splits.
#pragma once
#include <algorithm>

#include "mx4_common.h"

namespace rwkv7mi {

constexpr int MG_N = 256;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* mg_lds_ptr;

struct MgArgs {
  Mx4Prob p[MX4_MAXPROB];  // (ws: the scales in the products' order [superstep][column][16])
  int rows, O, I, NS;      // NS supersteps of 512 inputs
  int mt, nt, gm, gn;      // row / column tiles, XCD tile group
  int S, sps;              // K splits, supersteps of each
  int64_t ldp;             // partials [problem][split][row][ldp]
  float* part;
};

// A lane holds row n of a 32-row tile and, across a pair of column groups, runs of 8
// consecutive columns: column of group g, lane n: 64 (g / 2) + 8 (n / 4) + 4 (g % 2)
// + n % 4.  Rows of 128 bytes in LDS, whose 16-byte chunk c sits at c ^ key, the key
// from the lane n that reads the row: (n % 8) ^ (n / 8 % 2), which leaves 16-byte
// reads of one chunk a half wave free of bank conflicts on gfx950.
__device__ __forceinline__ int mg_key(int r) { return (r & 7) ^ ((r >> 3) & 1); }  // of x's row r
__device__ __forceinline__ int mg_wkey(int c) { return mg_key(4 * (c >> 3) + (c & 3)); }  // of W's column c

// XCD-aware tile number: workgroup L runs on XCD L % 8, which takes a run of the
// grouped tile order.  False: a padding tile.
__device__ __forceinline__ bool mg_tile(const MgArgs& B, int& tm, int& tn) {
  const int ngm = (B.mt + B.gm - 1) / B.gm, ngn = (B.nt + B.gn - 1) / B.gn;
  const int gsz = B.gm * B.gn, tiles = ngm * ngn * gsz;
  const int per = (tiles + 7) / 8;
  const int t = ((int)blockIdx.x % 8) * per + (int)blockIdx.x / 8;
  if (t >= tiles) return false;
  const int grp = t / gsz, gi = t % gsz;
  tm = grp / ngn * B.gm + gi / B.gn;
  tn = grp % ngn * B.gn + gi % B.gn;
  return tm < B.mt && tn < B.nt;
}

// 8 columns of a row from c0: bias and epilogue, before the rounding
template <typename T>
__device__ __forceinline__ void mg_finish8(const Mx4Prob& P, int64_t row, int c0, int O, bool vec, float (&v)[8]) {
  const int64_t oi = row * O + c0;
  const bool whole = vec && c0 + 8 <= O;
  const T* bp = static_cast<const T*>(P.bias);
  const T* rp = static_cast<const T*>(P.residual) + oi;
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = 0.f;
  if (P.epilogue == RWKV7MI_EPI_RESIDUAL) {
    if (whole) {
      ld8(rp, r);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c0 + e < O) r[e] = to_f32(rp[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (bp && c0 + e < O) v[e] += to_f32(bp[c0 + e]);
    if (P.epilogue == RWKV7MI_EPI_RELU2) v[e] = mx4_relu2(v[e]);
    v[e] += r[e];
  }
}

// 16-byte rows of y (and of the residual)
__device__ __forceinline__ bool mg_vec(const Mx4Prob& P, int O) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(P.y) |
                      (P.epilogue == RWKV7MI_EPI_RESIDUAL ? reinterpret_cast<uintptr_t>(P.residual) : 0);
  return O % 8 == 0 && !(a & 15);
}

// The tile's end.  Lane: row 32 i + n and, in group j, columns 64 (j / 2) + 16 a + 8 u
// + 4 (j % 2) .. +3, a = 0 .. 3.  The sums go through LDS (the stages are done with),
// two row tiles a wave at a time, and come back as whole rows: 32 lanes a row, 8
// columns each, whose bias stays in registers, stored past the caches, where they would
// push out operands (16384 x 4096 -> 16384 with 4-bit rows 700 -> 667 us, 1000 rows 52.6
// -> 50.3).  (Finished and stored from the MFMA layout, 32-byte pieces of 32 rows an
// instruction, the epilogue of the 4-bit rows took as long as half their main loop;
// rounded before LDS, with half the bytes there, 705 us.)
constexpr int MG_LDT = MG_N * 4 + 16;  // a staged row (the 16 bytes spread it over the banks)
constexpr int mg_staging(int mi) { return (mi < 2 ? 64 : 128) * MG_LDT; }

// cs: a factor per column of the tile, before the bias (in LDS; null: none).
template <int MI, int WC, bool SPLIT, typename T>
__device__ __forceinline__ void mg_epilogue(const MgArgs& B, const Mx4Prob& P, char* smem, const f32x16 (&acc)[MI][8 / WC],
                                            int m0, int n0, const float* cs) {
  constexpr int W = 2 * WC, RT = MI < 2 ? 1 : 2;  // waves; row tiles a wave and pass
  const int O = B.O, M = B.rows, nrow = min(64 * MI, M - m0);
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, u = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave / WC, wn = MG_N / WC * (wave % WC);
  const bool vec = mg_vec(P, O);
  const int epi = P.epilogue;
  const T *bias = static_cast<const T*>(P.bias), *res = static_cast<const T*>(P.residual);
  T* y = static_cast<T*>(P.y);
  float* part = SPLIT ? B.part + ((int64_t)blockIdx.y * B.S + blockIdx.z) * M * B.ldp : nullptr;
  // columns c0 + 8 l .. (one run), or, where rows do not start on 16 bytes, every 32nd from
  // l on, so that a store's lanes lie side by side (6319 x 1440 -> 7307, 4-bit rows, 114 -> 83 us)
  const bool whole = SPLIT || vec;
  const int step = whole ? 1 : 32, cl = whole ? 8 * (lane & 31) : lane & 31, c0 = n0 + cl;
  float bo[8], co[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    bo[e] = !SPLIT && bias && c0 + e * step < O ? to_f32(bias[c0 + e * step]) : 0.f;
    co[e] = cs ? cs[cl + e * step] : 1.f;
  }
#pragma unroll
  for (int p = 0; p < MI / RT; ++p) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < 8 / WC; ++j)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
          const f32x16 c = acc[RT * p + i][j];
          *reinterpret_cast<f32x4*>(smem + (32 * (RT * wr + i) + n) * MG_LDT +
                                    (wn + 64 * (j >> 1) + 16 * a + 8 * u + 4 * (j & 1)) * 4) =
              (f32x4){c[4 * a], c[4 * a + 1], c[4 * a + 2], c[4 * a + 3]};
        }
    __syncthreads();
    if (c0 >= O) continue;
    // four rows at a time: their LDS reads (and residuals) are in flight together;
    // staged row s is row s + 32 (MI - RT) (s / (32 RT)) + 32 RT p of the tile
    const auto finish = [&](auto run) {
      constexpr bool RUN = decltype(run)::value;
      for (int sb = 2 * wave + (lane >> 5); sb < 64 * RT; sb += 8 * W) {
        float v[4][8], w[4][8];
        int r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int s = sb + 2 * W * k;
          r[k] = s + 32 * (MI - RT) * (s / (32 * RT)) + 32 * RT * p;
          const float* at = reinterpret_cast<const float*>(smem + s * MG_LDT) + cl;
          if constexpr (RUN) {
            ld8(at, v[k]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = at[32 * e];
          }
        }
        if (!SPLIT && epi == RWKV7MI_EPI_RESIDUAL) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int64_t oi = (int64_t)(m0 + min(r[k], nrow - 1)) * O + c0;
            if constexpr (RUN) {
              ld8(res + oi, w[k]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[k][e] = c0 + 32 * e < O ? to_f32(res[oi + 32 * e]) : 0.f;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (r[k] >= nrow) continue;
          const int64_t row = m0 + r[k], oi = row * O + c0;
          if constexpr (SPLIT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] *= co[e];
            st8(part + row * B.ldp + c0, v[k]);
            continue;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[k][e] = v[k][e] * co[e] + bo[e];
          if (epi == RWKV7MI_EPI_RELU2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] = mx4_relu2(v[k][e]);
          } else if (epi == RWKV7MI_EPI_RESIDUAL) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[k][e] += w[k][e];
          }
          if constexpr (RUN) {
            u32x4 t;
            st8(reinterpret_cast<T*>(&t), v[k]);
            __builtin_nontemporal_store(t, reinterpret_cast<u32x4*>(y + oi));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c0 + 32 * e < O) y[oi + 32 * e] = from_f32<T>(v[k][e]);
          }
        }
      }
    };
    if (whole)
      finish(std::true_type{});
    else if constexpr (!SPLIT)
      finish(std::false_type{});
  }
}

// One thread: 8 columns of a row, the S partials in split order
template <typename T>
__global__ __launch_bounds__(256) void mg_reduce_kernel(const MgArgs B) {
  const Mx4Prob& P = B.p[blockIdx.y];
  const int cols = (int)(B.ldp / 8);
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= (int64_t)B.rows * cols) return;
  const int64_t row = t / cols;
  const int c0 = 8 * (int)(t % cols);
  if (c0 >= B.O) return;
  const int64_t zs = (int64_t)B.rows * B.ldp;
  const float* p = B.part + (int64_t)blockIdx.y * B.S * zs + row * B.ldp + c0;
  float v[8];
  ld8(p, v);
  for (int z = 1; z < B.S; ++z) {
    float a[8];
    ld8(p + z * zs, a);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += a[e];
  }
  const bool vec = mg_vec(P, B.O);
  mg_finish8<T>(P, row, c0, B.O, vec, v);
  T* y = static_cast<T*>(P.y) + row * B.O + c0;
  if (vec) {
    st8(y, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < B.O) y[e] = from_f32<T>(v[e]);
  }
}

static inline int64_t mg_up256(int64_t v) { return (v + 255) & ~(int64_t)255; }

// Tiles of an XCD group along one side: all up to 8, else the 4 to 8 that pad the
// side least (padding tiles leave some XCDs idle: 300 x 2560 -> 10240 with 4-bit rows,
// 5 x 40 tiles, 33.7 us in groups of 4 x 8 and 19.7 in 5 x 8).
static inline int mg_group(int n) {
  if (n <= 8) return n;
  int best = 8;
  for (int g = 7; g >= 4; --g)
    if ((n + g - 1) / g * g < (n + best - 1) / best * best) best = g;
  return best;
}

// Tile height (rows / 64) and K splits: the cheapest by an estimate in us, rounds of
// 256 workgroups (one a CU), each a start and an epilogue (ends) and its supersteps
// (step), slower with the chip busy, and for splits the second launch and the
// partials' traffic.
struct MgCost {
  double ends[3], ends_busy[3], step[3], step_busy[3];  // for 64, 128 and 256 rows
};
struct MgPlan {
  int mi, S;
  double us;
};
static inline MgPlan mg_plan(const MgCost& c, int nprob, int64_t rows, int64_t O, int64_t NS) {
  MgPlan p{1, 1, 1e30};
  for (int k = 0; k < 3; ++k) {
    const int mi = 1 << k;
    const int64_t tiles = nprob * ((rows + 64 * mi - 1) / (64 * mi)) * ((O + MG_N - 1) / MG_N);
    for (int64_t S = 1; S <= 16 && (S == 1 || tiles * S <= 512); ++S) {
      const int64_t sps = (NS + S - 1) / S;
      if (S > NS || (NS + sps - 1) / sps != S) continue;  // no empty split
      const int64_t rounds = (tiles * S + 255) / 256;
      const double busy = std::min(1.0, tiles * S / 256.0);
      const double split = S > 1 ? 6.0 + 0.4 * S + 8.0 * nprob * S * rows * O / 7e6 : 0.0;
      const double t = rounds * (c.ends[k] + c.ends_busy[k] * busy + (c.step[k] + c.step_busy[k] * busy) * sps) + split;
      if (t < p.us) p = MgPlan{mi, (int)S, t};
    }
  }
  return p;
}
static inline int64_t mg_part_bytes(const MgPlan& p, int nprob, int64_t rows, int64_t O) {
  return p.S > 1 ? mg_up256((int64_t)nprob * p.S * rows * ((O + 7) / 8 * 8) * 4) : 0;
}

// the launch's sizes (p is the caller's)
static inline void mg_sizes(MgArgs& a, const Mx4Batch& b, const MgPlan& pl) {
  a.rows = b.rows;
  a.O = b.O;
  a.I = b.I;
  a.NS = (b.I + 511) / 512;
  a.mt = (int)((b.rows + 64 * pl.mi - 1) / (64 * pl.mi));
  a.nt = (int)((b.O + MG_N - 1) / MG_N);
  a.gm = mg_group(a.mt);
  a.gn = mg_group(a.nt);
  a.S = pl.S;
  a.sps = (a.NS + pl.S - 1) / pl.S;
  a.ldp = (b.O + 7) / 8 * 8;
}
static inline dim3 mg_grid(const MgArgs& a, int nprob) {
  const int64_t tiles = (int64_t)((a.mt + a.gm - 1) / a.gm * a.gm) * ((a.nt + a.gn - 1) / a.gn * a.gn);
  return dim3((unsigned)((tiles + 7) / 8 * 8), (unsigned)nprob, (unsigned)a.S);
}
template <typename T>
static int mg_reduce(const MgArgs& a, int nprob, void* stream) {
  if (a.S == 1) return RWKV7MI_OK;
  const int64_t nthr = (int64_t)a.rows * (a.ldp / 8);
  hipLaunchKernelGGL(mg_reduce_kernel<T>, dim3((unsigned)((nthr + 255) / 256), (unsigned)nprob), dim3(256), 0,
                     as_stream(stream), a);
  return check_launch("mg_reduce_kernel");
}
// 32-bit offsets within a tile's 256 rows and columns and within the scales, 32-bit tile numbers
static inline bool mg_supported(int64_t rows, int64_t O, int64_t I) {
  const int64_t NS = (I + 511) / 512, tiles = (rows + 63) / 64 * ((O + MG_N - 1) / MG_N);
  return rows > 0 && 256 * 1024 * NS < (int64_t)BUF_OOB && 16 * NS * std::max(rows, O) < (int64_t)BUF_OOB &&
         rows <= INT32_MAX / 2 && O <= INT32_MAX / 2 && tiles < INT32_MAX / 64;
}

}  // namespace rwkv7mi
