// MXFP4 x MXFP4 products of many rows: y = epilogue(q(x) W^T + bias), q(x) the
// rows quantised by mx4_quantize_kernel.
//
// A 256-lane workgroup (four waves, one per SIMD) computes 16 MT rows x 256
// columns; wave w owns all rows x columns 64 w .. +63: MT x 4 tiles of
// v_mfma_scale_f32_16x16x128_f8f6f4, whose lane n + 16 q holds 32 inputs of one
// row (16 bytes of codes) and their scale byte.  W is the A operand, so a lane
// holds one row and, across a pair of column groups, 8 consecutive columns
// (columns permuted as 32 (g / 2) + 8 (n / 4) + 4 (g % 2) + n % 4): 16-byte
// stores.  K advances 256 inputs a step, two sub-steps of 128:
//  * W codes: global -> registers, one step ahead, straight from the row-major
//    layout (each wave reads its own columns only; no LDS);
//  * x codes: global -> LDS directly into three stages, two steps ahead; a row is
//    128 bytes whose 16-byte chunk c sits at c ^ key(row);
//  * scales: two steps (16 blocks, a superstep) at a time, global -> LDS, 16 bytes
//    a row and a column.  x's are laid out by the quantiser as [q][sub-step], so
//    one dword serves four sub-steps through the instruction's byte select; W's
//    come in their own order and are read a byte a lane and sub-step.
// x and its scales are padded to whole supersteps with zeros, so nothing past I
// counts (W's codes there are some finite value).
//
// The loads are spread over the MFMAs and waited for by count, and the one
// barrier a step lies between its sub-steps.  Where the tiles do not fill the
// chip K is split over workgroups and a second launch adds the fp32 partials.
#include <algorithm>

#include "mx4_common.h"

namespace rwkv7mi {

constexpr int MG_N = 256, MG_NST = 3;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* mg_lds_ptr;

struct MgArgs {
  Mx4Prob p[MX4_MAXPROB];
  int rows, O, I, NS;      // NS supersteps of 512 inputs
  int64_t ldws;            // bytes between the columns' scales
  int mt, nt, gm, gn;      // row / column tiles, XCD tile group
  int S, sps;              // K splits, supersteps of each
  int64_t ldp;             // partials [problem][split][row][ldp]
  float* part;
};

__device__ __forceinline__ int mg_key(int r) { return (r & 7) ^ ((r >> 3) & 1); }

__device__ __forceinline__ i32x8 mg_operand(u32x4 v) {
  return (i32x8){(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
}

template <int H>  // byte H of the B operand's scales
__device__ __forceinline__ f32x4 mg_mfma(u32x4 a, u32x4 b, f32x4 c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mg_operand(a), mg_operand(b), c, 4, 4, 0, sa, H, sb);
}

template <int N>
__device__ __forceinline__ void mg_wait() {  // vmcnt(N)
  __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | ((N >> 4) << 14));
}

// 8 columns of a row from c0: bias, epilogue, one rounding
template <typename T>
__device__ __forceinline__ void mg_store8(const Mx4Prob& P, int64_t row, int c0, int O, bool vec, float (&v)[8]) {
  const int64_t oi = row * O + c0;
  const bool whole = vec && c0 + 8 <= O;
  const T* bp = static_cast<const T*>(P.bias);
  const T* rp = static_cast<const T*>(P.residual) + oi;
  T* y = static_cast<T*>(P.y) + oi;
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
  if (whole) {
    st8(y, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c0 + e < O) y[e] = from_f32<T>(v[e]);
  }
}

// 16-byte rows of y (and of the residual)
__device__ __forceinline__ bool mg_vec(const Mx4Prob& P, int O) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(P.y) |
                      (P.epilogue == RWKV7MI_EPI_RESIDUAL ? reinterpret_cast<uintptr_t>(P.residual) : 0);
  return O % 8 == 0 && !(a & 15);
}

template <int MT, bool SPLIT, typename T>
__global__ __launch_bounds__(256, 1) void mx4_gemm_kernel(const MgArgs B) {
  constexpr int ROWS = 16 * MT, STAGE = ROWS * 128, SX = ROWS * 16, SW = MG_N * 16, NX = MT / 2;
  const Mx4Prob& P = B.p[blockIdx.y];
  const int O = B.O, M = B.rows, NS = B.NS;
  // XCD-aware tile number: workgroup L runs on XCD L % 8, which takes a run of the
  // grouped tile order (padding tiles exit)
  const int ngm = (B.mt + B.gm - 1) / B.gm, ngn = (B.nt + B.gn - 1) / B.gn;
  const int gsz = B.gm * B.gn, tiles = ngm * ngn * gsz;
  const int per = (tiles + 7) / 8;
  const int t = ((int)blockIdx.x % 8) * per + (int)blockIdx.x / 8;
  if (t >= tiles) return;
  const int grp = t / gsz, gi = t % gsz;
  const int tm = grp / ngn * B.gm + gi / B.gn, tn = grp % ngn * B.gn + gi % B.gn;
  if (tm >= B.mt || tn >= B.nt) return;
  const int m0 = tm * ROWS, n0 = tn * MG_N;

  extern __shared__ __align__(16) char smem[];  // x stages, then the scales of two supersteps
  char* const sxs = smem + MG_NST * STAGE;
  char* const sws = sxs + 2 * SX;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S0 = SPLIT ? (int)blockIdx.z * B.sps : 0;
  const int S1 = SPLIT ? min(NS, S0 + B.sps) : NS;
  const int s0 = 2 * S0, nsteps = 2 * (S1 - S0);

  // descriptors end at the tile's last row / column: past them zeros
  const int nrow = min(ROWS, M - m0), ncol = min(MG_N, O - n0);
  const int ldx = 256 * NS, ldw = B.I / 2;
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(P.xc + (int64_t)m0 * ldx, (uint32_t)(nrow * ldx));
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(P.wc + (int64_t)n0 * ldw, (uint32_t)((int64_t)ncol * ldw));
  const __amdgpu_buffer_rsrc_t xsr = make_rsrc(P.xs + (int64_t)m0 * 16 * NS, (uint32_t)(nrow * 16 * NS));
  const __amdgpu_buffer_rsrc_t wsr = make_rsrc(P.ws + (int64_t)n0 * B.ldws, (uint32_t)((int64_t)ncol * B.ldws));

  // x of step s: wave w, round u: rows 32 u + 8 w .. +7, lane l at row + l / 8,
  // chunk position l % 8
  int xo[NX];
#pragma unroll
  for (int u = 0; u < NX; ++u) {
    const int r = 32 * u + 8 * wave + (lane >> 3);
    xo[u] = r * ldx + 16 * ((lane & 7) ^ mg_key(r));
  }
  auto issue_x = [&](int s, int u) {
    const int so = s < nsteps ? 128 * (s0 + s) : (int)BUF_OOB, vo = xo[u];
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (mg_lds_ptr)(smem + s % MG_NST * STAGE + (32 * u + 8 * wave) * 128), 16,
                                             vo, so, 0, 0);
  };
  // W of step s: group j, sub-step h
  int wo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = 64 * wave + 32 * (j >> 1) + 8 * (n >> 2) + 4 * (j & 1) + (n & 3);
    wo[j] = col * ldw + 16 * q;
  }
  auto issue_w = [&](int s, int j, int h, u32x4 (&bw)[4][2]) {
    const int so = s < nsteps ? 128 * (s0 + s) + 64 * h : (int)BUF_OOB;
    bw[j][h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(wr, wo[j], so, 0));
  };
  // scales of superstep s: 64 rows (waves past the tile's rows repeat them) and the wave's 64 columns
  const int sr = 64 * (wave % (ROWS / 64)) + lane;
  const int sxo = sr * 16 * NS, swo = (64 * wave + lane) * (int)B.ldws;
  auto issue_s = [&](int s) {
    const int so = s < S1 - S0 ? 16 * (S0 + s) : (int)BUF_OOB;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xsr, (mg_lds_ptr)(sxs + (s & 1) * SX + 64 * (wave % (ROWS / 64)) * 16), 16, sxo,
                                             so, 0, 0);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(wsr, (mg_lds_ptr)(sws + (s & 1) * SW + 64 * wave * 16), 16, swo, so, 0, 0);
  };

  f32x4 acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int key = mg_key(n);
  const int ab0 = n * 128 + 16 * (q ^ key), ab1 = n * 128 + 16 * ((4 + q) ^ key);
  auto lda = [&](int st, int h, int i) {
    return *reinterpret_cast<const u32x4*>(smem + st * STAGE + (h ? ab1 : ab0) + 16 * i * 128);
  };
  auto ldsx = [&](int s, int i) { return *reinterpret_cast<const int*>(sxs + (s & 1) * SX + (16 * i + n) * 16 + 4 * q); };
  const int wcol = 64 * wave + 8 * (n >> 2) + (n & 3);
  auto ldsw = [&](int s, int h, int j) {
    return (int)*reinterpret_cast<const uint8_t*>(sws + (s & 1) * SW + (wcol + 32 * (j >> 1) + 4 * (j & 1)) * 16 + 4 * h + q);
  };

  u32x4 a[MT];         // x operands of a sub-step
  int sx[MT];          // x scales of the superstep
  int sw0[4], sw1[4];  // W scales of a sub-step, the next one's beside
  u32x4 bw0[4][2], bw1[4][2];

  // One sub-step: the MFMAs of the row tiles over `a`; a tile's operand of the next
  // sub-step is read as soon as its MFMAs are issued, so every read has a sub-step
  // to land.  `load(i)` issues the global loads of tile i.
  auto substep = [&](auto hc, const u32x4 (&bw)[4][2], const int (&sw)[4], int (&swn)[4], int st_n, int ss_n,
                     auto&& load) {
    constexpr int H = decltype(hc)::value;
#pragma unroll
    for (int j = 0; j < 4; ++j) swn[j] = ldsw(ss_n, (H + 1) & 3, j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mg_mfma<H>(bw[j][H & 1], a[i], acc[i][j], sw[j], sx[i]);
      a[i] = lda(st_n, (H + 1) & 1, i);
      if (H == 3) sx[i] = ldsx(ss_n, i);
      load(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  
  constexpr int WE = MT >= 16 ? 2 : 1, WP = MT >= 16 ? 1 : 8 / MT;  // W loads: every WE-th tile, WP a time
  auto w_loads = [&](int s, u32x4 (&bw)[4][2]) {
    return [&, s](int i) {
      if (i % WE == 0)
#pragma unroll
        for (int u = i / WE * WP; u < (i / WE + 1) * WP; ++u) issue_w(s, u & 3, u >> 2, bw);
    };
  };
  auto x_loads = [&](int s) {
    return [&, s](int i) {
      if (i % 2 == 0) issue_x(s, i / 2);
    };
  };

  // prologue: W and scales of step 0, x of steps 0 and 1 in flight
#pragma unroll
  for (int u = 0; u < 8; ++u) issue_w(0, u & 3, u >> 2, bw0);
  issue_s(0);
#pragma unroll
  for (int u = 0; u < NX; ++u) issue_x(0, u);
#pragma unroll
  for (int u = 0; u < NX; ++u) issue_x(1, u);
  mg_wait<NX>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int i = 0; i < MT; ++i) a[i] = lda(0, 0, i);
#pragma unroll
  for (int i = 0; i < MT; ++i) sx[i] = ldsx(0, i);
#pragma unroll
  for (int j = 0; j < 4; ++j) sw0[j] = ldsw(0, 0, j);

  // (separate zeros: sums that start as one shared value are moved from register to
  // register every turn of the loop, 1.5 moves an MFMA)
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) asm volatile("" : "+a"(acc[i][j]));
  for (int s = 0; s < nsteps; s += 2) {
    const int ss = s >> 1;
    // ---- step s: W of step s landed (x of step s + 1 may be pending)
    mg_wait<NX>();
    __builtin_amdgcn_sched_barrier(0);
    substep(std::integral_constant<int, 0>{}, bw0, sw0, sw1, s % MG_NST, ss, w_loads(s + 1, bw1));
    mg_wait<8>();  // x of step s + 1 landed; the barrier also puts every wave past step s - 1
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    issue_s(ss + 1);
    substep(std::integral_constant<int, 1>{}, bw0, sw1, sw0, (s + 1) % MG_NST, ss, x_loads(s + 2));
    // ---- step s + 1 (x of step s + 2 and the scales may be pending)
    mg_wait<NX + 2>();
    __builtin_amdgcn_sched_barrier(0);
    substep(std::integral_constant<int, 2>{}, bw1, sw0, sw1, (s + 1) % MG_NST, ss, w_loads(s + 2, bw0));
    mg_wait<8>();  // x of step s + 2 and the next superstep's scales landed
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    substep(std::integral_constant<int, 3>{}, bw1, sw1, sw0, (s + 2) % MG_NST, ss + 1, x_loads(s + 3));
  }
  mg_wait<0>();  // the trailing loads have landed before the waves exit

  // lane: row 16 i + n and, in groups 2 p and 2 p + 1, 8 columns from c0
  const bool vec = mg_vec(P, O);
  float* part = SPLIT ? B.part + ((int64_t)blockIdx.y * B.S + blockIdx.z) * M * B.ldp : nullptr;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int c0 = n0 + 64 * wave + 32 * p + 8 * q;
    if (c0 >= O) continue;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int row = m0 + 16 * i + n;
      if (row >= M) continue;
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = acc[i][2 * p][e];
        v[4 + e] = acc[i][2 * p + 1][e];
      }
      if constexpr (SPLIT)
        st8(part + (int64_t)row * B.ldp + c0, v);
      else
        mg_store8<T>(P, row, c0, O, vec, v);
    }
  }
}

// One thread: 8 columns of a row, the S partials in split order
template <typename T>
__global__ __launch_bounds__(256) void mx4_gemm_reduce_kernel(const MgArgs B) {
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
  mg_store8<T>(P, row, c0, B.O, mg_vec(P, B.O), v);
}

// W's scales with the rows of a ragged I padded to whole supersteps (1.0 there)
__global__ __launch_bounds__(256) void mx4_gemm_scales_kernel(const MgArgs B, uint8_t* out, int64_t each) {
  const int nb = B.I / MX4_BLOCK, ld = 16 * B.NS;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= (int64_t)B.O * ld) return;
  const int o = (int)(t / ld), b = (int)(t % ld);
  out[blockIdx.y * each + t] = b < nb ? B.p[blockIdx.y].ws[(int64_t)o * nb + b] : (uint8_t)127;
}

static int64_t up256(int64_t v) { return (v + 255) & ~(int64_t)255; }
struct MgPlan {
  int mt, S;                       // row tiles of 16 in a workgroup, K splits
  int64_t NS, codes, scales, pad, part;  // workspace bytes: x's codes and scales, padded W scales (a problem each), partials
};
static MgPlan mg_plan(int nprob, int64_t rows, int64_t O, int64_t I) {
  MgPlan p{};
  p.NS = (I + 511) / 512;
  p.codes = up256(rows * 256 * p.NS);
  p.scales = up256(rows * 16 * p.NS);
  p.pad = I % 512 ? up256(O * 16 * p.NS) : 0;
  p.mt = rows <= 64 ? 4 : rows <= 128 ? 8 : 16;
  p.S = 1;
  const int64_t tiles = nprob * ((rows + 16 * p.mt - 1) / (16 * p.mt)) * ((O + MG_N - 1) / MG_N);
  while (p.S < 8 && tiles * p.S * 2 <= 256 && p.NS / (p.S * 2) >= 1) p.S *= 2;
  const int64_t sps = (p.NS + p.S - 1) / p.S;
  p.S = (int)((p.NS + sps - 1) / sps);  // no empty split
  p.part = p.S > 1 ? up256((int64_t)nprob * p.S * rows * ((O + 7) / 8 * 8) * 4) : 0;
  return p;
}

bool mx4_gemm_supported(int64_t rows, int64_t O, int64_t I) {
  // 32-bit offsets within a tile's 256 rows and columns
  const int64_t NS = (I + 511) / 512, tiles = (rows + 63) / 64 * ((O + MG_N - 1) / MG_N);
  return rows > 0 && 256 * 256 * NS < (int64_t)BUF_OOB && rows <= INT32_MAX / 2 && O <= INT32_MAX / 2 &&
         tiles < INT32_MAX / 64;
}

int64_t mx4_gemm_workspace_bytes(int nprob, int64_t rows, int64_t O, int64_t I) {
  const MgPlan p = mg_plan(nprob, rows, O, I);
  return nprob * (p.codes + p.scales + p.pad) + p.part;
}

template <int MT, typename T>
static int mg_go(const MgArgs& a, int nprob, void* stream) {
  constexpr int lds = MG_NST * 16 * MT * 128 + 2 * (16 * MT + MG_N) * 16;
  const int64_t tiles = (int64_t)((a.mt + a.gm - 1) / a.gm * a.gm) * ((a.nt + a.gn - 1) / a.gn * a.gn);
  const dim3 grid((unsigned)((tiles + 7) / 8 * 8), (unsigned)nprob, (unsigned)a.S);
  static std::atomic<uint64_t> raised[2];
  auto launch = [&](auto kern, std::atomic<uint64_t>& done) {
    if (int rc = raise_dynamic_lds(reinterpret_cast<const void*>(kern), lds, done, "mx4_gemm_kernel")) return rc;
    hipLaunchKernelGGL(kern, grid, dim3(256), lds, as_stream(stream), a);
    return check_launch("mx4_gemm_kernel");
  };
  if (a.S == 1) return launch(&mx4_gemm_kernel<MT, false, T>, raised[0]);
  if (int rc = launch(&mx4_gemm_kernel<MT, true, T>, raised[1])) return rc;
  const int64_t nthr = (int64_t)a.rows * (a.ldp / 8);
  hipLaunchKernelGGL(mx4_gemm_reduce_kernel<T>, dim3((unsigned)((nthr + 255) / 256), (unsigned)nprob), dim3(256), 0,
                     as_stream(stream), a);
  return check_launch("mx4_gemm_reduce_kernel");
}

int mx4_gemm_run(const Mx4Batch& b, int nprob, int act_dtype, void* ws, void* stream) {
  const MgPlan pl = mg_plan(nprob, b.rows, b.O, b.I);
  MgArgs a{};
  a.rows = b.rows;
  a.O = b.O;
  a.I = b.I;
  a.NS = (int)pl.NS;
  a.ldws = pl.pad ? 16 * pl.NS : b.I / MX4_BLOCK;
  a.mt = (int)((b.rows + 16 * pl.mt - 1) / (16 * pl.mt));
  a.nt = (int)((b.O + MG_N - 1) / MG_N);
  a.gm = std::min(a.mt, 4);
  a.gn = std::min(a.nt, 8);
  a.S = pl.S;
  a.sps = (int)((pl.NS + pl.S - 1) / pl.S);
  a.ldp = (b.O + 7) / 8 * 8;
  uint8_t* at = static_cast<uint8_t*>(ws);
  const void* x[MX4_MAXPROB];
  uint8_t *xc[MX4_MAXPROB], *xs[MX4_MAXPROB];
  for (int i = 0; i < nprob; ++i) {
    a.p[i] = b.p[i];
    x[i] = b.p[i].x;
    a.p[i].xc = xc[i] = at;
    a.p[i].xs = xs[i] = at + pl.codes;
    at += pl.codes + pl.scales;
  }
  if (int rc = mx4_quantize_padded(nprob, x, b.rows, b.I, act_dtype, xc, xs, stream)) return rc;
  if (pl.pad) {
    const int64_t cells = (int64_t)b.O * 16 * pl.NS;
    hipLaunchKernelGGL(mx4_gemm_scales_kernel, dim3((unsigned)((cells + 255) / 256), (unsigned)nprob), dim3(256), 0,
                       as_stream(stream), a, at, pl.pad);
    if (int rc = check_launch("mx4_gemm_scales_kernel")) return rc;
    for (int i = 0; i < nprob; ++i) a.p[i].ws = at + i * pl.pad;
    at += nprob * pl.pad;
  }
  a.part = reinterpret_cast<float*>(at);
  const auto go = [&](auto t) {
    using T = decltype(t);
    return pl.mt == 4 ? mg_go<4, T>(a, nprob, stream) : pl.mt == 8 ? mg_go<8, T>(a, nprob, stream)
                                                                   : mg_go<16, T>(a, nprob, stream);
  };
  return act_dtype == RWKV7MI_BF16 ? go(__hip_bfloat16{}) : go(__half{});
}

}  // namespace rwkv7mi
