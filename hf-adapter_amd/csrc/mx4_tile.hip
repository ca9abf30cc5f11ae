// MXFP4 weights times many 16-bit rows: y = epilogue(x W^T + bias),
// fp16 / bf16 x.
//
// The tile of mx4_gemm.h with eight waves (two a SIMD, so that one's conversions and
// waits hide behind the other's MFMAs: 16384 x 4096 -> 16384 2.14 -> 1.98 ms) on
// v_mfma_f32_32x32x16: lane n + 32 u holds 8 inputs of a row.  K advances 64 inputs a
// step, four sub-steps; lane half u takes the block of inputs 32 u .. +31, 8 a sub-step,
// so a lane's scale holds for a step:
//  * x: global -> LDS directly, 128 bytes a row, a ring of NXS stages; lane n + 32 u reads
//    chunk 4 u + h in sub-step h;
//  * W codes: global -> LDS directly, 128 bytes (four steps) a column, two stages; a lane
//    reads 16 bytes a step, one dword a sub-step, which four conversions turn into its
//    operand during the sub-step before (a ring of 64-byte stages, 16384 x 4096 ->
//    16384: 2.04 ms);
//  * W's scales: 8 steps (a superstep) at a time, global -> LDS, 16 bytes a column; for
//    rows of scales that are not whole dwords (I % 128) from a copy that a pre-pass lays
//    out.  Columns are scaled by the largest scale of the workgroup's part of them
//    (mx4_common.h), which it reads first, while the ring fills, and the sums by its
//    factor (with the pre-pass at all sizes: 64 x 4096 -> 65536 76 us for 59, 1000 x
//    4096 -> 16384 1.6 us more, 4000 x 4096 -> 4096 4 less).
// A stage of x is read to the end in its step's third sub-step: one barrier there, and
// the loads a ring ahead go into the same stage; the barrier waits for the loads of the
// next step only, by count (with two stages every load had to land within a step: 64 x
// 16384 -> 4096 took 0.85 us a step).  Inputs past I are zeros of x (W's codes there are
// some finite value).  Where the tiles do not fill the chip K is split over workgroups
// and a second launch adds the partials.
//
// Bound by the MFMAs and the conversions beside them: 1000 x 4096 -> 16384 115 us in fp16,
// 110 in bf16, 1.17 and 1.22 PFLOP/s; a bare loop of these MFMAs on random operands runs
// at 1.68, a large library product of 16-bit operands at 1.11.
#include "mx4_gemm.h"

namespace rwkv7mi {

__device__ __forceinline__ f32x16 mt_mfma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mt_mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

constexpr int MT_WC = 4, MT_WAVES = 2 * MT_WC;
// x stages: what W's two leave room for, and W's loads, four steps ahead, are waited for
constexpr int mt_xstages(int mi) { return mi <= 2 ? 5 : 2; }
constexpr int mt_lds(int mi) {
  return std::max(mt_xstages(mi) * 64 * mi * 128 + 2 * MG_N * (128 + 16), mg_staging(mi));
}  // (then the columns' factors)
struct MtArgs {
  MgArgs g;
  int laid;  // p.ws: the pre-pass's copy, [superstep][column][16]
};
static_assert(mt_lds(1) + 4 * MG_N <= 163840 && mt_lds(2) + 4 * MG_N <= 163840 && mt_lds(4) + 4 * MG_N <= 163840,
              "LDS of a CU");

template <int MI, bool SPLIT, typename T>
__global__ __launch_bounds__(64 * MT_WAVES, 1) void mx4_tile_kernel(const MtArgs A) {
  const MgArgs& B = A.g;
  using V = typename Mx4Types<T>::V;
  constexpr int ROWS = 64 * MI, XB = ROWS * 128, WB = MG_N * 128, SB = MG_N * 16;  // bytes of a stage of x, W, scales
  constexpr int NXS = mt_xstages(MI);
  constexpr int NJ = 8 / MT_WC, RND = 8 * MT_WAVES;  // column groups of a wave; rows a round of loads
  constexpr int NX = ROWS / RND, NW = MG_N / RND;    // loads of a wave a stage of x, of W
  const Mx4Prob& P = B.p[blockIdx.y];
  const int M = B.rows, O = B.O, I = B.I, NS = B.NS;
  int tm, tn;
  if (!mg_tile(B, tm, tn)) return;
  const int m0 = tm * ROWS, n0 = tn * MG_N;

  extern __shared__ __align__(16) char smem[];  // the stages of x, W and (two) the scales
  char* const wst = smem + NXS * XB;
  char* const scl = wst + 2 * WB;
  float* const factor = reinterpret_cast<float*>(smem + mt_lds(MI));
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, u = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S0 = SPLIT ? (int)blockIdx.z * B.sps : 0;
  const int S1 = SPLIT ? min(NS, S0 + B.sps) : NS;
  const int s0 = 8 * S0, nsteps = min(8 * S1, (I + 63) / 64) - s0;  // (the last superstep may be short)

  // descriptors end at the tile's last row / column: past them zeros
  const int nrow = min(ROWS, M - m0), ncol = min(MG_N, O - n0);
  const int ldx = 2 * I, ldw = I / 2;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(static_cast<const char*>(P.x) + (int64_t)m0 * ldx, (uint32_t)(nrow * ldx));
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(P.wc + (int64_t)n0 * ldw, (uint32_t)(ncol * ldw));
  const int nb = I / MX4_BLOCK;
  const uint8_t* const ws = A.laid ? P.ws : P.ws + (int64_t)n0 * nb;
  const __amdgpu_buffer_rsrc_t wsr = make_rsrc(ws, (uint32_t)(A.laid ? NS * O * 16 : ncol * nb));

  // round v of a stage: rows RND v + 8 w .. +7 of x (W), lane l at row + l / 8, chunk
  // position l % 8
  const int lr = 8 * wave + (lane >> 3);
  auto issue_x = [&](int s, int st, int v) {
    const int r = RND * v + lr, c = (lane & 7) ^ mg_key(r);
    const int vo = 64 * (s0 + s) + 8 * c < I ? r * ldx + 16 * c : (int)BUF_OOB;
    const int so = s < nsteps ? 128 * (s0 + s) : (int)BUF_OOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (mg_lds_ptr)(smem + st * XB + (RND * v + 8 * wave) * 128), 16, vo, so, 0, 0);
  };
  auto issue_w = [&](int f, int v) {  // steps 4 f .. +3
    const int r = RND * v + lr, vo = r * ldw + 16 * ((lane & 7) ^ mg_wkey(r));
    const int so = 4 * f < nsteps ? 128 * (s0 / 4 + f) : (int)BUF_OOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (mg_lds_ptr)(wst + (f & 1) * WB + (RND * v + 8 * wave) * 128), 16, vo, so, 0,
                                             0);
  };
  auto issue_s = [&](int s) {  // scales of superstep s: 64 columns a wave of the first four
    if (wave >= MG_N / 64) return;
    const int at = A.laid ? 16 * ((S0 + s) * O + n0) : 16 * (S0 + s), so = s < S1 - S0 ? at : (int)BUF_OOB;
    const int vo = (64 * wave + lane) * (A.laid ? 16 : nb);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wsr, (mg_lds_ptr)(scl + (s & 1) * SB + 64 * wave * 16), 16, vo, so, 0, 0);
  };

  const int wm = 32 * MI * (wave / MT_WC), wn = MG_N / MT_WC * (wave % MT_WC);  // the wave's rows and columns in the tile
  const int wcol = 8 * (n >> 2) + (n & 3), key = mg_key(n);
  auto ld_x = [&](int st, int h, int i) {
    return *reinterpret_cast<const V*>(smem + st * XB + (wm + 32 * i + n) * 128 + 16 * ((4 * u + h) ^ key));
  };
  auto col = [&](int j) { return wn + 64 * (j >> 1) + 4 * (j & 1) + wcol; };
  auto ld_w = [&](int s, int j) {  // the lane's block of step s
    return *reinterpret_cast<const u32x4*>(wst + (s >> 2 & 1) * WB + col(j) * 128 + 16 * ((2 * (s & 3) + u) ^ key));
  };
  uint32_t emax[NJ];  // (of the lane's columns)
  auto ld_s = [&](int s, int j) {  // its scale byte
    const uint32_t e = *reinterpret_cast<const uint8_t*>(scl + (s >> 3 & 1) * SB + col(j) * 16 + 2 * (s & 7) + u);
    return mx4_run_byte<T>(e, emax[j]);
  };

  f32x16 acc[MI][NJ];
  V xa[2][MI], wa[2][NJ];     // operands of two sub-steps
  u32x4 wc[NJ], wcn[NJ];      // codes of this step and the next
  uint32_t sc[NJ], scn[NJ];   // their scale bytes

  // Sub-step H of step s (operand set H & 1): its MFMAs; the next sub-step's x operands
  // are read (from stage st) and its W operands made meanwhile, and in H = 3 load(l), l =
  // 0 .. NX - 1, issues x's loads.
  auto substep = [&](auto hc, int st, auto&& load) {
    constexpr int H = decltype(hc)::value, A = H & 1, HN = (H + 1) & 3, L = H == 3 ? NX : 0;
    constexpr int TILES = MI * NJ;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int k = NJ * i + j;
        acc[i][j] = mt_mfma(wa[A][j], xa[A][i], acc[i][j]);
        // x's reads over the first half, W's conversions over all of it
#pragma unroll
        for (int r = min(MI, k * 2 * MI / TILES); r < min(MI, (k + 1) * 2 * MI / TILES); ++r)
          xa[A ^ 1][r] = ld_x(st, HN, r);
        if (H == 3 && i == 0) wc[j] = wcn[j], sc[j] = scn[j];
#pragma unroll
        for (int r = k * NJ / TILES; r < (k + 1) * NJ / TILES; ++r) mx4_decode8(wc[r][HN], mx4_scale(sc[r]), wa[A ^ 1][r]);
#pragma unroll
        for (int l = k * L / TILES; l < (k + 1) * L / TILES; ++l) load(l);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  // every wave's operand reads, and all its loads but the newest NL, have landed, for all to see
  auto meet = [&](auto nl) {
    constexpr int NL = decltype(nl)::value;
    __builtin_amdgcn_s_waitcnt(0x0070 | (NL & 15) | (NL >> 4) << 14);  // vmcnt(NL), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  auto none = [](int) {};

  issue_s(0);
#pragma unroll
  for (int v = 0; v < 2 * NW; ++v) issue_w(v / NW, v % NW);
#pragma unroll
  for (int s = 0; s < NXS; ++s)
#pragma unroll
    for (int v = 0; v < NX; ++v) issue_x(s, s, v);
  {
    // the largest scale of column tid / 2, every other 8 bytes a thread
    const int c = tid >> 1, b0 = 16 * S0 + 8 * (tid & 1), be = min(16 * S1, nb);
    uint32_t m = 0;
    if (A.laid) {
      for (int s = S0; s < S1; ++s) {
        const uint2 d = *reinterpret_cast<const uint2*>(P.ws + 16 * ((int64_t)s * O + min(n0 + c, O - 1)) + 8 * (tid & 1));
        m = max(m, max(mx4_max4(d.x), mx4_max4(d.y)));
      }
    } else {
      const uint8_t* col = ws + (int64_t)min(c, ncol - 1) * nb;
#pragma unroll 4
      for (int s = S0; s < S1; ++s) {  // (past the end the last dword again)
        const int b = b0 + 16 * (s - S0);
        const uint32_t d0 = *reinterpret_cast<const uint32_t*>(col + min(b, be - 4));
        const uint32_t d1 = *reinterpret_cast<const uint32_t*>(col + min(b + 4, be - 4));
        m = max(m, max(mx4_max4(d0), mx4_max4(d1)));
      }
    }
    m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
    if (!(tid & 1)) factor[c] = mx4_run_factor<T>(m);
    __syncthreads();
  }
  meet(std::integral_constant<int, 0>{});
#pragma unroll
  for (int j = 0; j < NJ; ++j) emax[j] = mx4_factor_emax<T>(factor[col(j)]);
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    wc[j] = ld_w(0, j);
    sc[j] = ld_s(0, j);
    mx4_decode8(wc[j][0], mx4_scale(sc[j]), wa[0][j]);
  }
#pragma unroll
  for (int i = 0; i < MI; ++i) xa[0][i] = ld_x(0, 0, i);
  // (separate zeros: sums that start as one shared value are moved from register to
  // register every turn of the loop)
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
      asm volatile("" : "+a"(acc[i][j]));
    }
  int st = 0;  // the stage of x of step s
  for (int s = 0; s < nsteps; ++s) {
    substep(std::integral_constant<int, 0>{}, st, none);
    substep(std::integral_constant<int, 1>{}, st, none);
    substep(std::integral_constant<int, 2>{}, st, none);
    // x of step s read to its end, x of step s + 1 (and its codes and scales) there: of
    // the loads of NXS - 2 steps, x's at least, none is waited for
    meet(std::integral_constant<int, (NXS - 2) * NX>{});
    const int sn = st == NXS - 1 ? 0 : st + 1;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      wcn[j] = ld_w(s + 1, j);
      scn[j] = ld_s(s + 1, j);
    }
    if ((s & 7) == 0) issue_s((s >> 3) + 1);
    if ((s & 3) == 3) {  // a stage of W's last codes were read a step ago
#pragma unroll
      for (int v = 0; v < NW; ++v) issue_w(s / 4 + 2, v);
    }
    substep(std::integral_constant<int, 3>{}, sn, [&](int l) { issue_x(s + NXS, st, l); });
    st = sn;
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the trailing loads have landed before the waves exit

  mg_epilogue<MI, MT_WC, SPLIT, T>(B, P, smem, acc, m0, n0, factor);
}

// The pre-pass: the scales [superstep][column][16], 0 behind a column's end.  One thread
// a superstep of a column.
struct MtScales {
  const uint8_t* in[MX4_MAXPROB];
  u32x4* out[MX4_MAXPROB];
  int O, nb, NS;
};
__global__ __launch_bounds__(256) void mx4_tile_scales_kernel(const MtScales S) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= (int64_t)S.O * S.NS) return;
  const int o = (int)(t / S.NS), b0 = 16 * (int)(t % S.NS);
  const uint8_t* in = S.in[blockIdx.y] + (int64_t)o * S.nb;
  u32x4 v = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (b0 + i < S.nb) v[i >> 2] |= (uint32_t)in[b0 + i] << (8 * (i & 3));
  S.out[blockIdx.y][(int64_t)(b0 >> 4) * S.O + o] = v;
}

// Fitted to 19 shapes from 17 x 2048 -> 2048 to 7000 x 2048 -> 2048, every tile height and
// split timed, e.g. 1000 x 4096 -> 4096: 64 rows a tile 49.2 us, 128 rows 59.7, 256 rows
// in four splits 64.0; 4000 rows: 178, 136, 119; 64 x 16384 -> 4096: 64 rows in 16 splits
// 36.4, unsplit 154.
static const MgCost MX4_TILE_COST = {{1.0, 4.0, 5.5}, {0.0, 0.0, 3.5}, {4.6, 6.3, 9.5}, {0.9, 0.5, 3.5}};
static MgPlan mx4_tile_plan(int nprob, int64_t rows, int64_t O, int64_t I) {
  return mg_plan(MX4_TILE_COST, nprob, rows, O, (I + 511) / 512);
}
// (the plan's estimate, which compares tiles, leaves out some of what every call takes:
// over 22 shapes of 24 to 512 rows these sums choose the faster kernel)
double mx4_tile_us(int nprob, int64_t rows, int64_t O, int64_t I) {
  const MgPlan p = mx4_tile_plan(nprob, rows, O, I);
  return p.us + (p.S > 1 ? 5.0 : 4.0);
}
static bool mx4_tile_laid(int64_t I) { return I % (4 * MX4_BLOCK) != 0; }
static int64_t mx4_tile_scales(int64_t O, int64_t I) {
  return mx4_tile_laid(I) ? mg_up256(O * 16 * ((I + 511) / 512)) : 0;
}

bool mx4_tile_supported(int64_t rows, int64_t O, int64_t I) { return mg_supported(rows, O, I); }

int64_t mx4_tile_workspace_bytes(int nprob, int64_t rows, int64_t O, int64_t I) {
  return nprob * mx4_tile_scales(O, I) +
         mg_part_bytes(mx4_tile_plan(nprob, rows, O, I), nprob, rows, O);
}

template <int MI, typename T>
static int mt_go(const MtArgs& a, int nprob, void* stream) {
  constexpr int lds = mt_lds(MI) + 4 * MG_N;
  static std::atomic<uint64_t> raised[2];
  auto launch = [&](auto kern, std::atomic<uint64_t>& done) {
    if (int rc = raise_dynamic_lds(reinterpret_cast<const void*>(kern), lds, done, "mx4_tile_kernel")) return rc;
    hipLaunchKernelGGL(kern, mg_grid(a.g, nprob), dim3(64 * MT_WAVES), lds, as_stream(stream), a);
    if (int rc = check_launch("mx4_tile_kernel")) return rc;
    return mg_reduce<T>(a.g, nprob, stream);
  };
  return a.g.S == 1 ? launch(&mx4_tile_kernel<MI, false, T>, raised[0]) : launch(&mx4_tile_kernel<MI, true, T>, raised[1]);
}

int mx4_tile_run(const Mx4Batch& b, int nprob, int act_dtype, void* ws, void* stream) {
  const MgPlan pl = mx4_tile_plan(nprob, b.rows, b.O, b.I);
  const bool f16 = act_dtype == RWKV7MI_F16;
  MtArgs m{};
  MgArgs& a = m.g;
  mg_sizes(a, b, pl);
  m.laid = mx4_tile_laid(b.I);
  MtScales s{};
  s.O = b.O;
  s.nb = b.I / MX4_BLOCK;
  s.NS = a.NS;
  uint8_t* at = static_cast<uint8_t*>(ws);
  for (int i = 0; i < nprob; ++i) {
    a.p[i] = b.p[i];
    if (!m.laid) continue;
    s.in[i] = b.p[i].ws;
    s.out[i] = reinterpret_cast<u32x4*>(at);
    a.p[i].ws = at;
    at += mx4_tile_scales(b.O, b.I);
  }
  a.part = reinterpret_cast<float*>(at);
  if (m.laid) {
    const dim3 grid((unsigned)(((int64_t)b.O * a.NS + 255) / 256), (unsigned)nprob);
    hipLaunchKernelGGL(mx4_tile_scales_kernel, grid, dim3(256), 0, as_stream(stream), s);
    if (int rc = check_launch("mx4_tile_scales_kernel")) return rc;
  }
  const auto go = [&](auto t) {
    using T = decltype(t);
    return pl.mi == 1 ? mt_go<1, T>(m, nprob, stream) : pl.mi == 2 ? mt_go<2, T>(m, nprob, stream)
                                                                   : mt_go<4, T>(m, nprob, stream);
  };
  return f16 ? go(__half{}) : go(__hip_bfloat16{});
}

}  // namespace rwkv7mi
