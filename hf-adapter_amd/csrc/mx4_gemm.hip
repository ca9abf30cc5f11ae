// MXFP4 x MXFP4 products of many rows: y = epilogue(q(x) W^T + bias), q(x) the
// rows quantised by mx4_quantize_kernel.
//
// A 256-lane workgroup (four waves, one per SIMD) computes 64 MI rows x 256
// columns; wave w owns the rows 32 MI (w / 2) .. and the columns 128 (w % 2) ..:
// MI x 4 tiles of v_mfma_scale_f32_32x32x64_f8f6f4, whose lane n + 32 u holds 32
// inputs of one row (16 bytes of codes) and their scale byte.  (The 16x16x128 form
// does the same work in twice the instructions; one wave a SIMD could not issue
// them and the rest in time: 16384 x 4096 -> 16384, 37% of the MFMA cycles.)  W is
// the A operand, so a lane holds one row and, across a pair of column groups, 8
// consecutive columns (column of group g, lane n: 64 (g / 2) + 8 (n / 4) + 4 (g % 2)
// + n % 4): 16-byte stores.  K advances 256 inputs a step, four sub-steps of two
// blocks each:
//  * codes of x and W: global -> LDS directly, 128 bytes a row, two or three stages.  Whole
//    cache lines: 64-byte pieces straight into the operand registers stalled on
//    lines still on their way (16384 x 4096 -> 16384, 1.0 ms; without those loads
//    0.5).  A row's 16-byte chunk c sits at c ^ key, the key from the lane that
//    reads the row: (n % 8) ^ (n / 8 % 2), which leaves the reads free of bank
//    conflicts on gfx950.  Lane n + 32 u reads chunk 2 h + u in sub-step h;
//  * scales: two steps (16 blocks, a superstep) at a time, global -> LDS, 16 bytes
//    a row, in the order [u][step][sub-step], so that one dword serves a step's
//    four sub-steps through the instruction's byte select.  The quantiser's launch
//    writes both that way, the rows of a superstep side by side (16
//    bytes a row, rows apart, were a third of the kernel's L2 requests);
//  * x, and both scales, are padded to whole supersteps: x with zeros, so nothing
//    past I counts (W's codes there are some finite value).
//
// A sub-step's operands are read during the one before.  So a stage is read to the
// end in its step's third sub-step: one barrier there, and the loads a ring ahead go
// into the same stage, with a whole step or two to land.  Where the tiles do not
// fill the chip K is split over workgroups and a second launch adds the fp32
// partials.
//
// 16384 x 4096 -> 16384: 640 us with the quantiser, 3.4 PFLOP/s.  By its time over K (398 us
// at 2048 inputs, 622 at 4096, 1041 at 8192) the main loop takes 430 of them, 5.1 PFLOP/s of
// the 6.3 of a bare loop of these MFMAs on random codes; the rest is the start and the tiles'
// stores, 537 MB that all CUs write at about the same time.  Constant codes take 476 us (the
// bare loop 9.1 PFLOP/s): random ones run at a lower clock.
#include "mx4_gemm.h"

namespace rwkv7mi {

typedef int i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ i32x8 mg_operand(u32x4 v) {
  return (i32x8){(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}

template <int H>  // byte H of the scales
__device__ __forceinline__ f32x16 mg_mfma(u32x4 a, u32x4 b, f32x16 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mg_operand(a), mg_operand(b), c, 4, 4, H, sa, H, sb);
}

// Stages of codes: what LDS has room for (two with 64 and 128 rows too: 300 x 2560 ->
// 10240 22.2 us for 18.1, 200 x 4096 -> 16384 30.4 for 24.8).
constexpr int mg_stages(int mi) { return mi <= 2 ? 3 : 2; }
constexpr int mg_lds(int mi) {
  return std::max(mg_stages(mi) * (64 * mi + MG_N) * 128 + 2 * (64 * mi + MG_N) * 16, mg_staging(mi));
}
static_assert(mg_lds(1) <= 163840 && mg_lds(2) <= 163840 && mg_lds(4) <= 163840, "LDS of a CU");

template <int MI, bool SPLIT, typename T>
__global__ __launch_bounds__(256, 1) void mx4_gemm_kernel(const MgArgs B) {
  constexpr int ROWS = 64 * MI, XB = ROWS * 128, STAGE = XB + MG_N * 128, NST = mg_stages(MI);
  constexpr int SX = ROWS * 16, SB = SX + MG_N * 16, NX = 2 * MI;  // scale bytes; x loads a wave and step
  const Mx4Prob& P = B.p[blockIdx.y];
  const int M = B.rows, O = B.O, NS = B.NS;
  int tm, tn;
  if (!mg_tile(B, tm, tn)) return;
  const int m0 = tm * ROWS, n0 = tn * MG_N;

  extern __shared__ __align__(16) char smem[];  // the stages (x, W), the scales of two supersteps (x, W)
  char* const scl = smem + NST * STAGE;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 31, u = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S0 = SPLIT ? (int)blockIdx.z * B.sps : 0;
  const int S1 = SPLIT ? min(NS, S0 + B.sps) : NS;
  const int s0 = 2 * S0, nsteps = 2 * (S1 - S0);

  // descriptors end at the tile's last row / column: past them zeros
  const int nrow = min(ROWS, M - m0), ncol = min(MG_N, O - n0);
  const int ldx = 256 * NS, ldw = B.I / 2;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(P.xc + (int64_t)m0 * ldx, (uint32_t)(nrow * ldx));
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(P.wc + (int64_t)n0 * ldw, (uint32_t)(ncol * ldw));
  const __amdgpu_buffer_rsrc_t xsr = make_rsrc(P.xs, (uint32_t)(NS * M * 16));
  const __amdgpu_buffer_rsrc_t wsr = make_rsrc(P.ws, (uint32_t)(NS * O * 16));

  // codes of step s into stage st, round v: rows 32 v + 8 w .. +7 of x (W), lane l at row + l / 8,
  // chunk position l % 8
  const int lr = 8 * wave + (lane >> 3);
  auto issue_x = [&](int s, int st, int v) {
    const int r = 32 * v + lr, vo = r * ldx + 16 * ((lane & 7) ^ mg_key(r));
    const int so = s < nsteps ? 128 * (s0 + s) : (int)BUF_OOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (mg_lds_ptr)(smem + st * STAGE + (32 * v + 8 * wave) * 128), 16, vo, so, 0,
                                             0);
  };
  auto issue_w = [&](int s, int st, int v) {
    const int r = 32 * v + lr, vo = r * ldw + 16 * ((lane & 7) ^ mg_wkey(r));
    const int so = s < nsteps ? 128 * (s0 + s) : (int)BUF_OOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, (mg_lds_ptr)(smem + st * STAGE + XB + (32 * v + 8 * wave) * 128), 16, vo,
                                             so, 0, 0);
  };
  // scales of superstep s: 64 rows of x (waves past the tile's rows repeat them), 64 columns
  const int xw = wave % MI;
  auto issue_s = [&](int s) {
    const bool ok = s < S1 - S0;
    const int xo = ok ? 16 * ((S0 + s) * M + m0 + 64 * xw) : (int)BUF_OOB;
    const int wo = ok ? 16 * ((S0 + s) * O + n0 + 64 * wave) : (int)BUF_OOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xsr, (mg_lds_ptr)(scl + (s & 1) * SB + 64 * xw * 16), 16, 16 * lane, xo, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wsr, (mg_lds_ptr)(scl + (s & 1) * SB + SX + 64 * wave * 16), 16, 16 * lane, wo,
                                             0, 0);
  };

  const int wm = 32 * MI * (wave >> 1), wn = 128 * (wave & 1);  // the wave's rows and columns in the tile
  const int wcol = 8 * (n >> 2) + (n & 3), key = mg_key(n);
  auto ldx_op = [&](int st, int h, int i) {
    return *reinterpret_cast<const u32x4*>(smem + st * STAGE + (wm + 32 * i + n) * 128 + 16 * ((2 * h + u) ^ key));
  };
  auto ldw_op = [&](int st, int h, int j) {
    return *reinterpret_cast<const u32x4*>(smem + st * STAGE + XB + (wn + 64 * (j >> 1) + 4 * (j & 1) + wcol) * 128 +
                                           16 * ((2 * h + u) ^ key));
  };
  auto ldx_sc = [&](int s, int i) {
    return *reinterpret_cast<const int*>(scl + (s >> 1 & 1) * SB + (wm + 32 * i + n) * 16 + 8 * u + 4 * (s & 1));
  };
  auto ldw_sc = [&](int s, int j) {
    return *reinterpret_cast<const int*>(scl + (s >> 1 & 1) * SB + SX + (wn + 64 * (j >> 1) + 4 * (j & 1) + wcol) * 16 +
                                         8 * u + 4 * (s & 1));
  };

  f32x16 acc[MI][4];
  u32x4 xa[2][MI], wa[2][4];           // operands of two sub-steps
  int sx[MI], sw[4], sxn[MI], swn[4];  // scales of this step and the next

  // Sub-step H of step s (operand set H & 1): its MFMAs, the reads of the next
  // sub-step's operands (from stage st) over the first three quarters, and load(l) for l in L0 .. L1 - 1
  // spread over them.
  constexpr int LOADS = NX + 8, LCUT = LOADS / 2;  // the loads of a step: before and behind the cut
  auto substep = [&](auto hc, int s, int st, auto&& load, int L0, int L1) {
    constexpr int H = decltype(hc)::value, A = H & 1, HN = (H + 1) & 3;
    constexpr int TILES = MI * 4, READS = MI + 4, Q = TILES * 3 / 4;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = 4 * i + j;
        acc[i][j] = mg_mfma<H>(wa[A][j], xa[A][i], acc[i][j], sw[j], sx[i]);
        const int r0 = min(READS, k * READS / Q), r1 = min(READS, (k + 1) * READS / Q);
#pragma unroll
        for (int r = r0; r < r1; ++r) {  // W's first: every MFMA of the first row tile takes one
          if (r < 4)
            wa[A ^ 1][r] = ldw_op(st, HN, r);
          else
            xa[A ^ 1][r - 4] = ldx_op(st, HN, r - 4);
          if (H == 3) {
            if (r < 4)
              swn[r] = ldw_sc(s + 1, r);
            else
              sxn[r - 4] = ldx_sc(s + 1, r - 4);
          }
        }
#pragma unroll
        for (int l = L0 + k * (L1 - L0) / TILES; l < L0 + (k + 1) * (L1 - L0) / TILES; ++l) load(l);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  auto loads = [&](int s, int st) {
    return [&, s, st](int l) {
      if (l < NX)
        issue_x(s, st, l);
      else
        issue_w(s, st, l - NX);
    };
  };
  // every wave's operand reads, and all its loads but the newest NL, have landed, for all to see
  auto meet = [&](auto nl) {
    constexpr int NL = decltype(nl)::value;
    __builtin_amdgcn_s_waitcnt(0x0070 | (NL & 15) | (NL >> 4) << 14);  // vmcnt(NL), lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  issue_s(0);
#pragma unroll
  for (int l = 0; l < (NST - 1) * LOADS + LCUT; ++l)  // (step 0 issues the rest)
    loads(l / LOADS, l / LOADS)(l % LOADS);
  meet(std::integral_constant<int, (NST - 2) * LOADS + LCUT>{});
#pragma unroll
  for (int j = 0; j < 4; ++j) wa[0][j] = ldw_op(0, 0, j), sw[j] = ldw_sc(0, j);
#pragma unroll
  for (int i = 0; i < MI; ++i) xa[0][i] = ldx_op(0, 0, i), sx[i] = ldx_sc(0, i);
  // (separate zeros: sums that start as one shared value are moved from register to
  // register every turn of the loop, 1.5 moves an MFMA)
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
      asm volatile("" : "+a"(acc[i][j]));
    }
  int st = 0;  // the stage of step s
  for (int s = 0; s < nsteps; ++s) {
    const int sn = st == NST - 1 ? 0 : st + 1, sp = st == 0 ? NST - 1 : st - 1;
    substep(std::integral_constant<int, 0>{}, s, st, loads(s + NST - 1, sp), LCUT, LOADS);
    substep(std::integral_constant<int, 1>{}, s, st, loads(s, st), 0, 0);
    substep(std::integral_constant<int, 2>{}, s, st, loads(s, st), 0, 0);
    // step s read to its end, step s + 1 (and its scales) there: of the loads NST - 2
    // steps further none is waited for
    meet(std::integral_constant<int, (NST - 2) * LOADS>{});
    if ((s & 1) == 0) issue_s((s >> 1) + 1);
    substep(std::integral_constant<int, 3>{}, s, sn, loads(s + NST, st), 0, LCUT);
    st = sn;
#pragma unroll
    for (int i = 0; i < MI; ++i) sx[i] = sxn[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) sw[j] = swn[j];
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the trailing loads have landed before the waves exit

  mg_epilogue<MI, 2, SPLIT, T>(B, P, smem, acc, m0, n0, nullptr);
}

// Fitted to 18 shapes from 200 x 4096 -> 16384 to 7000 x 2048 -> 2048, every tile height
// and split timed, e.g. 1000 x 4096 -> 4096: 64 rows a tile 24.3 us, 128 rows 28.7, 256
// rows in two splits 38.2; 4000 rows: 78.5, 60.5, 54.9; 1500 x 16384 -> 2048: 128 rows
// in two splits 60.0, unsplit 71.0, 64 rows unsplit 61.8.
static const MgCost MX4_GEMM_COST = {{0.4, 3.4, 6.8}, {1.6, 0.0, 0.0}, {1.6, 1.8, 2.2}, {0.0, 0.4, 1.4}};
static MgPlan mx4_gemm_plan(int nprob, int64_t rows, int64_t O, int64_t I) {
  return mg_plan(MX4_GEMM_COST, nprob, rows, O, (I + 511) / 512);
}
// workspace bytes: x's codes and scales, W's scales (a problem each)
static int64_t mx4_gemm_codes(int64_t rows, int64_t I) { return mg_up256(rows * 256 * ((I + 511) / 512)); }
static int64_t mx4_gemm_scales(int64_t rows, int64_t I) { return mg_up256(rows * 16 * ((I + 511) / 512)); }

bool mx4_gemm_supported(int64_t rows, int64_t O, int64_t I) { return mg_supported(rows, O, I); }

int64_t mx4_gemm_workspace_bytes(int nprob, int64_t rows, int64_t O, int64_t I) {
  return nprob * (mx4_gemm_codes(rows, I) + mx4_gemm_scales(rows, I) + mx4_gemm_scales(O, I)) +
         mg_part_bytes(mx4_gemm_plan(nprob, rows, O, I), nprob, rows, O);
}

template <int MI, typename T>
static int mg_go(const MgArgs& a, int nprob, void* stream) {
  constexpr int lds = mg_lds(MI);
  static std::atomic<uint64_t> raised[2];
  auto launch = [&](auto kern, std::atomic<uint64_t>& done) {
    if (int rc = raise_dynamic_lds(reinterpret_cast<const void*>(kern), lds, done, "mx4_gemm_kernel")) return rc;
    hipLaunchKernelGGL(kern, mg_grid(a, nprob), dim3(256), lds, as_stream(stream), a);
    if (int rc = check_launch("mx4_gemm_kernel")) return rc;
    return mg_reduce<T>(a, nprob, stream);
  };
  return a.S == 1 ? launch(&mx4_gemm_kernel<MI, false, T>, raised[0]) : launch(&mx4_gemm_kernel<MI, true, T>, raised[1]);
}

int mx4_gemm_run(const Mx4Batch& b, int nprob, int act_dtype, void* ws, void* stream) {
  const MgPlan pl = mx4_gemm_plan(nprob, b.rows, b.O, b.I);
  MgArgs a{};
  mg_sizes(a, b, pl);
  uint8_t* at = static_cast<uint8_t*>(ws);
  uint8_t *xc[MX4_MAXPROB], *xs[MX4_MAXPROB], *wsc[MX4_MAXPROB];
  for (int i = 0; i < nprob; ++i) {
    a.p[i] = b.p[i];
    a.p[i].xc = xc[i] = at;
    a.p[i].xs = xs[i] = at + mx4_gemm_codes(b.rows, b.I);
    a.p[i].ws = wsc[i] = xs[i] + mx4_gemm_scales(b.rows, b.I);
    at = wsc[i] + mx4_gemm_scales(b.O, b.I);
  }
  if (int rc = mx4_quantize_padded(b, nprob, act_dtype, xc, xs, wsc, stream)) return rc;
  a.part = reinterpret_cast<float*>(at);
  const auto go = [&](auto t) {
    using T = decltype(t);
    return pl.mi == 1 ? mg_go<1, T>(a, nprob, stream) : pl.mi == 2 ? mg_go<2, T>(a, nprob, stream)
                                                                   : mg_go<4, T>(a, nprob, stream);
  };
  return act_dtype == RWKV7MI_BF16 ? go(__hip_bfloat16{}) : go(__half{});
}

}  // namespace rwkv7mi
