// Recurrent-state slot copies for the serving state pool
// (docs/integrations/RWKV7_STATE_CACHE_ABI.md:52-133: layer-major pools
// S_pool [L, capacity, H, N, N], xpa / xpf [L, capacity, D], v_first
// [capacity, A]; gather / scatter / clone / reset of scheduled slots).
//
// One launch moves rows of every layer: row r of layer l goes from
//   src + l * src_layer_stride + src_rows[r] * src_row_stride
// to
//   dst + l * dst_layer_stride + dst_rows[r] * dst_row_stride
// (strides in bytes; a null row-index array means the identity), skipping
// rows whose active flag is 0, and writing zeros when src is null.  A row is
// row_bytes long (a multiple of 16, 16-byte aligned): each thread moves 16
// bytes per pass with plain vector loads and stores.  Grid: (row chunks,
// rows, layers).  Byte copies, no arithmetic.
#include "common.h"

namespace rwkv7mi {

struct SlotCopy {
  const char* src;
  char* dst;
  const int64_t* src_rows;
  const int64_t* dst_rows;
  const uint8_t* active;
  int64_t src_layer, dst_layer, src_row, dst_row;
  int64_t row16;  // 16-byte units per row
};

__global__ __launch_bounds__(256) void slot_copy_kernel(const SlotCopy C) {
  const int64_t r = blockIdx.y;
  const int64_t l = blockIdx.z;
  if (C.active && !C.active[r]) return;
  const int64_t sr = C.src_rows ? C.src_rows[r] : r;
  const int64_t dr = C.dst_rows ? C.dst_rows[r] : r;
  uint4* d = reinterpret_cast<uint4*>(C.dst + l * C.dst_layer + dr * C.dst_row);
  const uint4* s = C.src ? reinterpret_cast<const uint4*>(C.src + l * C.src_layer + sr * C.src_row) : nullptr;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < C.row16; i += (int64_t)gridDim.x * 256)
    d[i] = s ? s[i] : make_uint4(0u, 0u, 0u, 0u);
}

// Rows of several tensors moved by one index in one launch:
//   dst[o][d(r)] = the old src[o][s(r)]   for every outer index o and every r,
// as if all sources were read before any destination is written, so rows may
// trade places in place; s(r) out of range (-1) writes zeros (or bytes of 0xff:
// NaN in fp16, bf16 and fp32), d(r) out of range nothing, and a row onto itself is
// left alone.
//
// A workgroup takes a window of the row's bytes of one tensor and outer index
// for all rows: it gathers the rows that move into a list, loads all their
// windows into registers, and stores them behind a barrier.  What it reads
// it alone writes, so no launch but this one is needed, and a source with many
// destinations comes from memory once.  The window shrinks as the rows grow
// (THREADS x LOADS units of 16 bytes over the rows, a power of two).
//
// HBM-bound.  The stores go past the caches: behind ordinary ones (in brackets)
// the same moves of states that the caches do not hold take up to 1.3 times as
// long.  us for the fp32 states of the 7.2B model (33.5 MB a row): 8 chats of 4
// beams in place, 0.99 GB, 183 [189]; one row to 8, 0.31 GB, 50 [64]; two rows to
// four each in new tensors, 0.34 GB, 51 [67]; the 2.9B model's fp16 pool of 33, 9
// rows moved and 5 made zero, 0.25 GB, 48 [58]; 4 rows of the 0.1B model 4.2 [4.3].
// (Rows trading places in pairs, states of 9 to 537 MB: 0 to 9% more than behind
// ordinary stores, with a pass over the states behind the move up to 2%.  In an
// earlier build, behind ordinary stores, 4 loads a lane: 8% less to 13% more, the
// largest moves losing; 16: up to a third more.)
namespace {

constexpr int RW_TENSORS = 24;   // of a launch
constexpr int RW_LIST = 192;     // indices that travel with the launch
constexpr int RW_FEW = 64;       // rows of the small workgroup
constexpr int RW_MOST = 2048;    // rows of the large one (windows of 64 bytes)

struct RwTensor {
  const char* src;
  char* dst;
  int64_t src_outer, dst_outer, src_row, dst_row;  // strides in bytes
  uint32_t units, windows;                         // of a row, units of `unit` bytes
  int64_t outer;
  int unit, same;                                  // same: in place
};

struct RwArgs {
  RwTensor t[RW_TENSORS];
  uint32_t first[RW_TENSORS + 1];  // the tensor's first workgroup
  int n, rows, log_window, split;  // split: rows of a workgroup
  int64_t src_rows, dst_rows;
  const int64_t *src_index, *dst_index;  // on the device (null: the list, or the identity)
  int listed_src, listed_dst;
  uint32_t fill;  // what a source out of range writes
  int src_list[RW_LIST], dst_list[RW_LIST];
};

template <typename V>
__device__ __forceinline__ void rw_hold(V& v) {  // v is in its registers here
  if constexpr (sizeof(V) == 16)
    asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));
  else
    asm volatile("" : "+v"(v));
}
template <typename V>
__device__ __forceinline__ V rw_filled(uint32_t f) {
  if constexpr (sizeof(V) == 16)
    return make_uint4(f, f, f, f);
  else
    return f;
}

template <int THREADS, int LOADS, typename V, typename HELD>
__device__ __forceinline__ void rw_window(const RwTensor& t, int64_t o, uint32_t w0, int log_window, int n, const int* src,
                                          const int* dst, uint32_t fill) {
  const int tid = threadIdx.x, mask = (1 << log_window) - 1;
  HELD r[LOADS];
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int j = tid + THREADS * u, k = j >> log_window;
    const uint32_t c = w0 + (uint32_t)(j & mask);
    r[u] = rw_filled<HELD>(fill);
    if (k < n && c < t.units && src[k] >= 0)
      r[u] = static_cast<HELD>(reinterpret_cast<const V*>(t.src + o * t.src_outer + src[k] * t.src_row)[c]);
  }
#pragma unroll
  for (int u = 0; u < LOADS; ++u) rw_hold(r[u]);
  __syncthreads();
#pragma unroll
  for (int u = 0; u < LOADS; ++u) {
    const int j = tid + THREADS * u, k = j >> log_window;
    const uint32_t c = w0 + (uint32_t)(j & mask);
    if (k >= n || c >= t.units) continue;
    V* p = reinterpret_cast<V*>(t.dst + o * t.dst_outer + dst[k] * t.dst_row) + c;
    if constexpr (sizeof(V) == 16)
      __builtin_nontemporal_store(u32x4{r[u].x, r[u].y, r[u].z, r[u].w}, reinterpret_cast<u32x4*>(p));
    else
      *p = static_cast<V>(r[u]);
  }
}

}  // namespace

template <int THREADS, int LOADS, int ROWS>
__global__ __launch_bounds__(THREADS) void rows_move_kernel(const RwArgs A) {
  __shared__ int src[ROWS], dst[ROWS], moving;
  int f = 0;
  while (f + 1 < A.n && blockIdx.x >= A.first[f + 1]) ++f;
  const RwTensor& t = A.t[f];
  const uint32_t at = blockIdx.x - A.first[f];
  const int64_t o = at / t.windows;
  const uint32_t w = at % t.windows;
  if (threadIdx.x == 0) moving = 0;
  __syncthreads();
  const int r1 = min(A.rows, ((int)blockIdx.y + 1) * A.split);
  for (int r = (int)blockIdx.y * A.split + threadIdx.x; r < r1; r += THREADS) {
    const int64_t s = A.src_index ? A.src_index[r] : A.listed_src ? A.src_list[r] : r;
    const int64_t d = A.dst_index ? A.dst_index[r] : A.listed_dst ? A.dst_list[r] : r;
    if (d >= 0 && d < A.dst_rows && !(t.same && s == d)) {
      const int p = atomicAdd(&moving, 1);
      src[p] = s >= 0 && s < A.src_rows ? (int)s : -1;
      dst[p] = (int)d;
    }
  }
  __syncthreads();
  const int n = moving;
  if (n == 0) return;
  if (t.unit == 16)
    rw_window<THREADS, LOADS, uint4, uint4>(t, o, w << A.log_window, A.log_window, n, src, dst, A.fill);
  else if (t.unit == 4)
    rw_window<THREADS, LOADS, uint32_t, uint32_t>(t, o, w << A.log_window, A.log_window, n, src, dst, A.fill);
  else
    rw_window<THREADS, LOADS, uint8_t, uint32_t>(t, o, w << A.log_window, A.log_window, n, src, dst, A.fill);
}

}  // namespace rwkv7mi

using namespace rwkv7mi;

extern "C" int rwkv7mi_slot_copy(const void* src, int64_t src_layer_stride, int64_t src_row_stride,
                                 const int64_t* src_rows, void* dst, int64_t dst_layer_stride,
                                 int64_t dst_row_stride, const int64_t* dst_rows, const uint8_t* active,
                                 int64_t nrows, int64_t row_bytes, int64_t nlayers, void* stream) {
  if (nrows < 0 || nlayers < 0 || row_bytes <= 0 || row_bytes % 16)
    return fail(RWKV7MI_EINVAL, "slot_copy: row_bytes must be a positive multiple of 16");
  if (nrows == 0 || nlayers == 0) return RWKV7MI_OK;
  if (!dst) return fail(RWKV7MI_EINVAL, "slot_copy: null destination");
  if (nrows > 65535 || nlayers > 65535) return fail(RWKV7MI_EINVAL, "slot_copy: at most 65535 rows and layers");
  if ((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | (uintptr_t)src_layer_stride |
       (uintptr_t)src_row_stride | (uintptr_t)dst_layer_stride | (uintptr_t)dst_row_stride) & 15)
    return fail(RWKV7MI_EINVAL, "slot_copy: pointers and strides must be 16-byte aligned");
  SlotCopy c{reinterpret_cast<const char*>(src), reinterpret_cast<char*>(dst), src_rows, dst_rows, active,
             src_layer_stride, dst_layer_stride, src_row_stride, dst_row_stride, row_bytes / 16};
  const int64_t chunks = std::min<int64_t>((c.row16 + 255) / 256, 64);
  hipLaunchKernelGGL(slot_copy_kernel, dim3((unsigned)chunks, (unsigned)nrows, (unsigned)nlayers), dim3(256), 0,
                     as_stream(stream), c);
  return check_launch("slot_copy_kernel");
}

extern "C" int rwkv7mi_rows_move(int n, const rwkv7mi_rows* tensors, int64_t src_rows, int64_t dst_rows, int64_t nrows,
                                 const int64_t* src_index, const int64_t* dst_index, const int64_t* src_list,
                                 const int64_t* dst_list, int flags, void* stream) {
  const std::string w("rows_move");
  if (n < 0 || n > RW_TENSORS || (n && !tensors)) return fail(RWKV7MI_EINVAL, w + ": at most 24 tensors");
  if (nrows < 0 || src_rows < 0 || dst_rows < 0 || src_rows > INT32_MAX || dst_rows > INT32_MAX)
    return fail(RWKV7MI_EINVAL, w + ": bad rows");
  if ((src_list || dst_list) && nrows > RW_LIST) return fail(RWKV7MI_EINVAL, w + ": at most 192 indices in host lists");
  if ((src_list && src_index) || (dst_list && dst_index))
    return fail(RWKV7MI_EINVAL, w + ": a list and a device index of the same rows");
  if (flags & ~3) return fail(RWKV7MI_EINVAL, w + ": unknown flags");
  const bool disjoint = flags & RWKV7MI_ROWS_DISJOINT;
  RwArgs a{};
  a.fill = flags & RWKV7MI_ROWS_POISON ? ~0u : 0u;
  bool same = false;
  for (int i = 0; i < n; ++i) {
    const rwkv7mi_rows& t = tensors[i];
    if (t.row_bytes < 0 || t.outer < 0) return fail(RWKV7MI_EINVAL, w + ": bad shape");
    if (nrows == 0 || t.row_bytes == 0 || t.outer == 0) continue;
    if ((!t.src && src_rows) || !t.dst) return fail(RWKV7MI_EINVAL, w + ": null pointer");
    RwTensor& q = a.t[a.n++];
    q.src = static_cast<const char*>(t.src);
    q.dst = static_cast<char*>(t.dst);
    q.src_outer = t.src_outer_stride;
    q.dst_outer = t.dst_outer_stride;
    q.src_row = t.src_row_stride;
    q.dst_row = t.dst_row_stride;
    q.same = t.src == t.dst;
    if (q.same && (q.src_outer != q.dst_outer || q.src_row != q.dst_row))
      return fail(RWKV7MI_EINVAL, w + ": a tensor in place keeps its strides");
    same |= q.same;
    const uint64_t align = (uint64_t)reinterpret_cast<uintptr_t>(t.src) | (uint64_t)reinterpret_cast<uintptr_t>(t.dst) |
                           (uint64_t)t.src_outer_stride | (uint64_t)t.dst_outer_stride | (uint64_t)t.src_row_stride |
                           (uint64_t)t.dst_row_stride | (uint64_t)t.row_bytes;
    q.unit = align % 16 == 0 ? 16 : align % 4 == 0 ? 4 : 1;
    if (t.row_bytes / q.unit > INT32_MAX) return fail(RWKV7MI_EINVAL, w + ": a row is too long");
    q.units = (uint32_t)(t.row_bytes / q.unit);
    q.outer = t.outer;
  }
  if (a.n == 0) return RWKV7MI_OK;
  if (same && !disjoint && nrows > RW_MOST)
    return fail(RWKV7MI_EINVAL, w + ": at most 2048 rows trade places in place");
  // rows that may trade places stay in one workgroup
  const bool few = !same || disjoint || nrows <= RW_FEW;
  a.rows = (int)nrows;
  a.split = few ? RW_FEW : RW_MOST;
  const int64_t units = few ? 256 * 8 : 1024 * 8, held = std::min<int64_t>(nrows, a.split);
  while ((units >> (a.log_window + 1)) >= held) ++a.log_window;
  uint64_t blocks = 0;
  for (int i = 0; i < a.n; ++i) {
    a.first[i] = (uint32_t)blocks;
    a.t[i].windows = (uint32_t)(((uint64_t)a.t[i].units + (1u << a.log_window) - 1) >> a.log_window);
    if (a.t[i].outer > INT32_MAX ||
        (blocks += (uint64_t)a.t[i].outer * a.t[i].windows) > UINT32_MAX / (few ? 256u : 1024u)) return fail(RWKV7MI_EINVAL, w + ": too large");
  }
  a.first[a.n] = (uint32_t)blocks;
  a.src_rows = src_rows;
  a.dst_rows = dst_rows;
  a.src_index = src_index;
  a.dst_index = dst_index;
  a.listed_src = src_list != nullptr;
  a.listed_dst = dst_list != nullptr;
  for (int64_t r = 0; r < nrows && (src_list || dst_list); ++r) {
    if (src_list) a.src_list[r] = (int)std::max<int64_t>(std::min<int64_t>(src_list[r], INT32_MAX), -2);
    if (dst_list) a.dst_list[r] = (int)std::max<int64_t>(std::min<int64_t>(dst_list[r], INT32_MAX), -2);
  }
  const int64_t chunks = (nrows + a.split - 1) / a.split;
  if (chunks > 65535) return fail(RWKV7MI_EINVAL, w + ": too many rows");
  const dim3 grid((unsigned)blocks, (unsigned)chunks);
  if (few)
    hipLaunchKernelGGL((rows_move_kernel<256, 8, RW_FEW>), grid, dim3(256), 0, as_stream(stream), a);
  else
    hipLaunchKernelGGL((rows_move_kernel<1024, 8, RW_MOST>), grid, dim3(1024), 0, as_stream(stream), a);
  return check_launch("rows_move_kernel");
}
