// The seam between two transformer blocks in one pass over the rows:
//     h = residual_scale * residual + gate * rms(y) * post_weight      (the new residual stream)
//     n = rms(h) * pre_weight                                          (input of the next block)
// with rms(v) = v / sqrt(mean(v^2) + eps), and its backward pass.  y is the output of the block
// that has just finished (an MLP or a mixture of experts).
//
// Both passes are bound by HBM: forward reads y and residual and writes h and n (4 values per
// element), backward reads dh, dn, y, residual and writes dy, dresidual (6 values; h and the
// normalised rows are recomputed in fp32 from the saved reciprocal norms, because a weight
// gradient summed from an h that was rounded to 16 bits would carry that rounding).  Nothing is
// read from memory twice; reductions and all arithmetic are fp32.
//
// Many rows go through the ring kernels: a block walks its share of the rows, whole rows arrive in
// shared memory by bulk copies a few rows ahead, so that the two reductions of a row (a barrier
// each) never leave HBM idle.  With a block per row and plain loads the same arithmetic reached
// 59 % (forward) and 39 % (backward) of the copy rate at 4096 bf16 columns.  Few rows take the
// plain kernels.
#include <cuda_runtime.h>

#include <mutex>

#include "tnx_elem.cuh"
#include "tnx_internal.h"
#include "tnx_ptx.cuh"

namespace tnx {

namespace {

struct NormParams {
  int rows, cols;
  int gate_form;
  float alpha, eps;
  long long ld_y, ld_res, ld_gate, ld_dh, ld_dn;  // row pitches in elements; the others are `cols`
  const void *y, *res, *post, *pre, *gate;
  void *h, *n;
  float* stats;  // [rows][2]: reciprocal norms of y and of h
  // backward
  const void *dh, *dn;
  void *dy, *dres, *dgate;  // dgate: [rows] (token form) or [rows][cols] (full form), weight type
  float* partial;           // [grid][sums][cols]: column sums for post, pre and a channel gate
  int sums;
  // ring kernels
  int depth;                // rows in flight
  int edge, inner;          // rows at either end of a tensor that are copied in part, and those between
  int* status;
  unsigned long long timeout_ns;
};

constexpr int kMaxCols = 16384;
// Threads of a row at most, by the values each of them holds: 256 with up to 16 values (two or
// three blocks per SM), then 512; single elements 640.  LED rows take a warp more, so that 608 threads
// of 8 values (640 of two short vectors: five fp32 rows leave room for one block only) and 480 of
// more leave each thread the registers it needs.
__host__ __device__ constexpr int max_threads(int vec, int nv, bool led = false) {
  if (led) return vec * nv > 8 ? 480 : nv == 2 ? 640 : 608;
  return vec == 1 ? 640 : vec * nv <= 16 ? 256 : 512;
}
// Threads of a block of a ring kernel at most, and blocks per SM that its registers are limited for.
__host__ __device__ constexpr int ring_threads(int vec, int nv, bool led) { return max_threads(vec, nv, led) + (led ? 32 : 0); }
__host__ __device__ constexpr int ring_blocks(int vec, int nv, bool led, bool backward) {
  return max_threads(vec, nv, led) > 256 ? 1 : backward ? 2 : 3;
}

// Sums of two values over the `threads` threads of a row.  `slot` alternates between calls so
// that one barrier per call is enough.  Every thread of the block takes part.
__device__ __forceinline__ float2 row_sum(float a, float b, float2* smem, int threads, int tid) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (threads == 32) return make_float2(a, b);
  if ((tid & 31) == 0) smem[tid >> 5] = make_float2(a, b);
  __syncthreads();
  const int warps = threads >> 5;
  const int lane = tid & 31;
  float2 v = lane < warps ? smem[lane] : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

// The gate of one vector of a row (1 where there is none).
template <typename W, int VEC>
__device__ __forceinline__ void load_gate(const NormParams& p, int row, int col, float (&g)[VEC]) {
  const W* gate = static_cast<const W*>(p.gate);
  if (p.gate_form == TNX_GATE_CHANNEL) {
    elem::load<W, VEC>(gate + col, g);
  } else if (p.gate_form == TNX_GATE_FULL) {
    elem::load<W, VEC>(gate + row * p.ld_gate + col, g);
  } else {
    const float v = p.gate_form == TNX_GATE_TOKEN ? elem::to_float(gate[row * p.ld_gate]) : 1.f;
#pragma unroll
    for (int i = 0; i < VEC; ++i) g[i] = v;
  }
}

// blockDim = (threads of a row, rows of the block).  Vector v of a row belongs to thread
// v % threads; a thread owns up to NV vectors.
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(max_threads(VEC, NV), 1) norm_forward_kernel(const NormParams p) {
  __shared__ float2 sums[2][32];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int row = blockIdx.x * blockDim.y + threadIdx.y;
  const bool live = row < p.rows;
  float2* slot0 = sums[0] + threadIdx.y * (threads >> 5);
  float2* slot1 = sums[1] + threadIdx.y * (threads >> 5);
  const T* y_row = static_cast<const T*>(p.y) + row * p.ld_y;
  const T* r_row = static_cast<const T*>(p.res) + row * p.ld_res;

  float y[NV][VEC], h[NV][VEC];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (tid + i * threads) * VEC;
    if (live && col < p.cols) {
      elem::load<T, VEC>(y_row + col, y[i]);
      elem::load<T, VEC>(r_row + col, h[i]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) y[i][j] = h[i][j] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) ss += y[i][j] * y[i][j];
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  const float r1 = rsqrtf(row_sum(ss, 0.f, slot0, threads, tid).x * inv_cols + p.eps);
  ss = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (tid + i * threads) * VEC;
    if (live && col < p.cols) {
      float w[VEC], g[VEC];
      elem::load<W, VEC>(static_cast<const W*>(p.post) + col, w);
      load_gate<W, VEC>(p, row, col, g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        h[i][j] = p.alpha * h[i][j] + g[j] * (y[i][j] * r1 * w[j]);
        ss += h[i][j] * h[i][j];
      }
    }
  }
  const float r2 = rsqrtf(row_sum(ss, 0.f, slot1, threads, tid).x * inv_cols + p.eps);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (tid + i * threads) * VEC;
    if (col < p.cols) {
      float w[VEC], n[VEC];
      elem::load<W, VEC>(static_cast<const W*>(p.pre) + col, w);
#pragma unroll
      for (int j = 0; j < VEC; ++j) n[j] = h[i][j] * r2 * w[j];
      const long long at = static_cast<long long>(row) * p.cols + col;
      elem::store<T, VEC>(static_cast<T*>(p.h) + at, h[i]);
      elem::store<T, VEC>(static_cast<T*>(p.n) + at, n);
    }
  }
  if (p.stats != nullptr && tid == 0) {
    p.stats[2 * static_cast<long long>(row)] = r1;
    p.stats[2 * static_cast<long long>(row) + 1] = r2;
  }
}

// Backward.  With a = y r1, b = a post, u = dn pre (all per row, <.> the mean over columns):
//   dh' = dh + r2 (u - h r2^2 <u h>)            total gradient of h
//   dresidual = alpha dh',  dgate = dh' b,  dpre = dn h r2,  dpost = gate dh' a
//   v = gate dh' post,  dy = r1 (v - a <v a>)
// A block walks rows blockIdx.x, blockIdx.x + gridDim.x, ... and keeps the column sums of its
// rows in registers; norm_column_sums adds the blocks' sums in a fixed order.
template <typename T, typename W, int VEC, int NV>
__global__ void __launch_bounds__(max_threads(VEC, NV), 1) norm_backward_kernel(const NormParams p) {
  __shared__ float2 sums[2][32];
  const int tid = threadIdx.x, threads = blockDim.x;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  float c_post[NV][VEC], c_pre[NV][VEC], c_gate[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) c_post[i][j] = c_pre[i][j] = c_gate[i][j] = 0.f;

  for (int row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const long long at = static_cast<long long>(row) * p.cols;
    const float r1 = p.stats[2 * static_cast<long long>(row)];
    const float r2 = p.stats[2 * static_cast<long long>(row) + 1];
    const T* y_row = static_cast<const T*>(p.y) + row * p.ld_y;
    const T* r_row = static_cast<const T*>(p.res) + row * p.ld_res;
    const T* dh_row = static_cast<const T*>(p.dh) + row * p.ld_dh;
    const T* dn_row = static_cast<const T*>(p.dn) + row * p.ld_dn;
    float a[NV][VEC], h[NV][VEC], d[NV][VEC], u[NV][VEC];
    float s_uh = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (tid + i * threads) * VEC;
      if (col < p.cols) {
        elem::load<T, VEC>(y_row + col, a[i]);
        elem::load<T, VEC>(r_row + col, h[i]);
        elem::load<T, VEC>(dh_row + col, d[i]);
        elem::load<T, VEC>(dn_row + col, u[i]);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[i][j] = h[i][j] = d[i][j] = u[i][j] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (tid + i * threads) * VEC;
      if (col < p.cols) {
        float post[VEC], pre[VEC], g[VEC];
        elem::load<W, VEC>(static_cast<const W*>(p.post) + col, post);
        elem::load<W, VEC>(static_cast<const W*>(p.pre) + col, pre);
        load_gate<W, VEC>(p, row, col, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          a[i][j] *= r1;
          h[i][j] = p.alpha * h[i][j] + g[j] * (a[i][j] * post[j]);
          c_pre[i][j] += u[i][j] * (h[i][j] * r2);
          u[i][j] *= pre[j];
          s_uh += u[i][j] * h[i][j];
        }
      }
    }
    const float k = row_sum(s_uh, 0.f, sums[0], threads, tid).x * inv_cols * r2 * r2;
    float s_va = 0.f, s_g = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (tid + i * threads) * VEC;
      if (col < p.cols) {
        float post[VEC], g[VEC], out[VEC], dg[VEC];
        elem::load<W, VEC>(static_cast<const W*>(p.post) + col, post);
        load_gate<W, VEC>(p, row, col, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float dh = d[i][j] + r2 * (u[i][j] - h[i][j] * k);
          out[j] = p.alpha * dh;
          dg[j] = dh * (a[i][j] * post[j]);
          const float db = g[j] * dh;
          c_post[i][j] += db * a[i][j];
          c_gate[i][j] += dg[j];
          s_g += dg[j];
          d[i][j] = db * post[j];
          s_va += d[i][j] * a[i][j];
        }
        elem::store<T, VEC>(static_cast<T*>(p.dres) + at + col, out);
        if (p.gate_form == TNX_GATE_FULL) elem::store<W, VEC>(static_cast<W*>(p.dgate) + at + col, dg);
      }
    }
    const float2 s = row_sum(s_va, s_g, sums[1], threads, tid);
    const float m = s.x * inv_cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (tid + i * threads) * VEC;
      if (col < p.cols) {
        float out[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = r1 * (d[i][j] - a[i][j] * m);
        elem::store<T, VEC>(static_cast<T*>(p.dy) + at + col, out);
      }
    }
    if (p.gate_form == TNX_GATE_TOKEN && tid == 0) static_cast<W*>(p.dgate)[row] = elem::from_float<W>(s.y);
  }
  float* mine = p.partial + static_cast<long long>(blockIdx.x) * p.sums * p.cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (tid + i * threads) * VEC;
    if (col < p.cols) {
      elem::store<float, VEC>(mine + col, c_post[i]);
      elem::store<float, VEC>(mine + p.cols + col, c_pre[i]);
      if (p.sums == 3) elem::store<float, VEC>(mine + 2 * static_cast<long long>(p.cols) + col, c_gate[i]);
    }
  }
}

// ------------------------------------------------------------------------------------ ring kernels

constexpr int kMaxDepth = 4;
constexpr int kAbort = 0x401;
struct RingCtrl {
  uint64_t full[kMaxDepth];
  float2 sums[2][32];
  int abort;
};
constexpr int kCtrlBytes = 768;
static_assert(sizeof(RingCtrl) <= kCtrlBytes, "control block too large");

// Shared memory for one row of one source: the row, moved by up to 15 bytes, in whole 16 bytes.
__host__ __device__ constexpr uint32_t ring_row_bytes(int cols, int size) { return (cols * size + 15 + 15) / 16 * 16; }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// A barrier of the whole block that warps may come to from different places, and whether `ok` held for
// every thread.
__device__ __forceinline__ bool block_barrier(bool ok = true) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.and.pred q, 0, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(ok))
      : "memory");
  return all != 0;
}

// Sums of N values over the block, and whether `ok` held for every thread.  `levels`: so many times
// two warps (blockDim.x is up to 32 << levels).
template <int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float2* smem, int levels, bool& ok) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if ((tid & 31) == 0) smem[tid >> 5] = make_float2(v[0], v[N - 1]);
  ok = block_barrier(ok);
  const int warps = blockDim.x >> 5, lane = tid & ((1 << levels) - 1);
  const float2 all = lane < warps ? smem[lane] : make_float2(0.f, 0.f);
  v[0] = all.x;
  v[N - 1] = N > 1 ? all.y : all.x;
  for (int o = 1 << levels >> 1; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
}

// The rows a block walks: blockIdx.x, blockIdx.x + gridDim.x, ...  Row number i of them lies in slot
// i % depth, one part of the slot per source.  A bulk copy starts and ends on 16-byte boundaries, so
// a row is copied from the boundary at or before its first byte to the one at or after its last.
// Only a tensor's first and last rows (one each, or as many as start within 15 bytes of an end) could
// be read past its ends that way: of those the copy brings what lies between two boundaries inside
// them, the bytes before and behind follow by ordinary loads (the whole of a last row by ordinary
// loads made its block 10 to 40 us late).
// MOVED: rows may start anywhere (otherwise all start on 16-byte boundaries), but all rows of a block
// equally far behind a boundary: the grid is a multiple of the rows after which that comes back.
// (Working the distance out for each row cost the thread that issues the copies, and with it the
// block, about a microsecond a row.)
constexpr int kMaxSources = 5;
// The part of a row that its bulk copy brings, in bytes from the boundary at or before the row's first
// byte; `shift`: the row's own distance from there.
struct CopyPart {
  uint32_t from, to;
};
__host__ __device__ constexpr CopyPart copy_part(uint32_t shift, uint32_t row_bytes, bool first, bool last) {
  const uint32_t from = first && shift > 0 ? 16u : 0u, to = (shift + row_bytes + (last ? 0u : 15u)) & ~15u;
  return {from, to > from ? to : from};
}
// Rows at either end of a tensor that lie within 15 bytes of it.  (Pitches below a row's length, 0 among
// them, only come here where all rows start and end on boundaries and are copied whole.)
inline int edge_rows(long long pitch_bytes) {
  return pitch_bytes < 1 || pitch_bytes > 14 ? 1 : 14 / static_cast<int>(pitch_bytes) + 1;
}
template <bool MOVED>
struct Ring {
  RingCtrl* ctrl;
  char* slots;  // (shared memory)
  int sources, depth, rows;
  uint32_t slot_bytes;
  const char* src[kMaxSources];
  long long pitch[kMaxSources];  // bytes
  uint32_t row_bytes[kMaxSources], offset[kMaxSources];
  uint32_t shift[kMaxSources];  // bytes from the boundary to a row's start
  int edge, inner;  // as in NormParams
  int row, slot;  // where the block is
  uint32_t phase;

  __device__ __forceinline__ Ring(char* smem, const NormParams& p)
      : ctrl(reinterpret_cast<RingCtrl*>(smem)), slots(smem + kCtrlBytes), sources(0), depth(p.depth), rows(p.rows),
        slot_bytes(0), edge(p.edge), inner(p.inner), row(blockIdx.x), slot(0), phase(0) {}
  template <typename E>
  __device__ __forceinline__ void add(const void* base, long long ld, int cols) {
    src[sources] = static_cast<const char*>(base);
    pitch[sources] = ld * static_cast<long long>(sizeof(E));
    row_bytes[sources] = static_cast<uint32_t>(cols * sizeof(E));
    offset[sources] = slot_bytes;
    shift[sources] =
        MOVED ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src[sources] + row * pitch[sources]) & 15) : 0u;
    slot_bytes += ring_row_bytes(cols, sizeof(E));
    ++sources;
  }
  // Source k's copy of row r.
  __device__ __forceinline__ CopyPart part(int k, long long r, bool first) const {
    return copy_part(shift[k], row_bytes[k], MOVED && first, MOVED && r >= edge + inner);
  }
  // One thread; first: the row is one of the tensors' first.
  __device__ __forceinline__ void issue(long long r, int to, bool first) {
    if (r >= rows) return;
    const uint32_t bar = ptx::smem_u32(&ctrl->full[to]);
    const uint32_t at = ptx::smem_u32(slots) + to * slot_bytes;
    uint32_t total = 0;
#pragma unroll
    for (int k = 0; k < kMaxSources; ++k)
      if (k < sources) total += part(k, r, first).to - part(k, r, first).from;
    ptx::mbar_arrive_expect_tx(bar, total);
#pragma unroll
    for (int k = 0; k < kMaxSources; ++k)
      if (k < sources) {
        const CopyPart c = part(k, r, first);
        if (c.to > c.from)
          bulk_load(at + offset[k] + c.from, src[k] + r * pitch[k] - shift[k] + c.from, c.to - c.from, bar);
      }
  }
  __device__ __forceinline__ void start() {
    if (threadIdx.x == 0) {
      for (int d = 0; d < depth; ++d) ptx::mbar_init(ptx::smem_u32(&ctrl->full[d]), 1);
      ctrl->abort = 0;
      ptx::fence_mbar_init();
      // (there are more blocks than rows at an end: only a block's own first row can be one of the first)
      for (int d = 0; d < depth; ++d) issue(row + static_cast<long long>(d) * gridDim.x, d, d == 0 && row < edge);
    }
    __syncthreads();
  }
  // The block's row is in its slot (false: it did not come in time).
  __device__ __forceinline__ bool wait(uint64_t limit_ns) {
    const bool ok = ptx::mbar_wait(ptx::smem_u32(&ctrl->full[slot]), phase, &ctrl->abort, limit_ns);
    if (!MOVED || static_cast<unsigned>(row - edge) < static_cast<unsigned>(inner)) return ok;
    // (all threads come here together; a row is a whole number of 2-byte pieces, and there are at most 15
    // bytes before and 15 behind)
#pragma unroll
    for (int k = 0; k < kMaxSources; ++k)
      if (k < sources) {
        const uint32_t moved = shift[k];
        const CopyPart c = part(k, row, row < edge);
        const uint32_t before = c.from > moved ? c.from - moved : 0u, behind = c.to > moved ? c.to - moved : 0u;
        const char* from = src[k] + row * pitch[k];
        char* to = slots + static_cast<size_t>(slot) * slot_bytes + offset[k] + moved;
        uint32_t b = threadIdx.x * 2;
        if (b < before && b < row_bytes[k]) *reinterpret_cast<uint16_t*>(to + b) = *reinterpret_cast<const uint16_t*>(from + b);
        b += behind;
        if (b < row_bytes[k]) *reinterpret_cast<uint16_t*>(to + b) = *reinterpret_cast<const uint16_t*>(from + b);
      }
    block_barrier();
    return ok;
  }
  // Byte offset of source k's row in the slots.
  __device__ __forceinline__ uint32_t at(int k) const { return slot * slot_bytes + offset[k] + shift[k]; }
  // Nobody reads the row's slot any more: it takes the row `depth` rounds ahead.
  __device__ __forceinline__ void refill() {
    if (threadIdx.x == 0) issue(row + static_cast<long long>(depth) * gridDim.x, slot, false);
  }
  __device__ __forceinline__ void next() {
    row += gridDim.x;
    if (++slot == depth) {
      slot = 0;
      phase ^= 1u;
    }
  }
  // A wait gave up: copies that are still in flight land before shared memory is given back.
  __device__ __forceinline__ void give_up(int* status) {
    if (threadIdx.x == 0 && status != nullptr) atomicCAS(status, 0, kAbort);
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
};

// The columns of a thread: vector n of VEC columns starts at first + n * step, and is the thread's if
// that is before limit.
struct Columns {
  int first, step, limit;
};
// Rows that do not start on 16-byte boundaries (an odd number of columns) are still read and written in
// whole vectors where every tensor has its rows moved alike (LED): `head` elements, then vectors, then
// a tail shorter than a vector.  Head and tail belong to a warp of their own, an element per lane: it
// runs the same row loop with VEC = NV = 1 and meets the other warps at the barriers.  A block only
// walks rows with one head (the grid is a multiple of the rows after which it comes back), so its
// threads keep their columns.  (Masking the first and the last vector instead made the warps that hold
// them late to every barrier: 55 us against 49, 8192 x 2049 bf16 forward, before the other steps.)
struct Led {
  int head, tail;
  bool edge;  // this thread is of the head's and the tail's warp
  __device__ __forceinline__ Led(int cols, int vec)
      : head(static_cast<int>(blockIdx.x * static_cast<long long>(cols) % vec)), edge(threadIdx.x >= blockDim.x - 32) {
    head = head == 0 ? 0 : vec - head < cols ? vec - head : cols;
    tail = (cols - head) % vec;
  }
  __device__ __forceinline__ Columns edges(int cols) const {
    const int lane = threadIdx.x & 31;
    return {lane < head ? lane : lane < head + tail ? cols - tail + lane - head : cols, 0, cols};
  }
  __device__ __forceinline__ Columns vectors(int cols, int vec) const {
    return {head + static_cast<int>(threadIdx.x) * vec, static_cast<int>(blockDim.x - 32) * vec, cols - tail};
  }
};
// Weights and column sums start on a 16-byte boundary whatever the rows do.
template <typename W, int VEC, bool LED>
__device__ __forceinline__ elem::Pack<W, VEC> column_pack(const W* at) {
  if constexpr (LED) {
    elem::Pack<W, VEC> raw;
#pragma unroll
    for (int j = 0; j < VEC; ++j) raw.v[j] = at[j];
    return raw;
  } else {
    return *reinterpret_cast<const elem::Pack<W, VEC>*>(at);
  }
}
template <typename W, int VEC, bool LED>
__device__ __forceinline__ void column_load(const W* at, float (&out)[VEC]) {
  const elem::Pack<W, VEC> raw = column_pack<W, VEC, LED>(at);
#pragma unroll
  for (int j = 0; j < VEC; ++j) out[j] = elem::to_float(raw.v[j]);
}
template <int VEC, bool LED>
__device__ __forceinline__ void column_store(float* at, const float (&in)[VEC]) {
  if constexpr (LED) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) at[j] = in[j];
  } else {
    elem::store<float, VEC>(at, in);
  }
}

// Weights that every row meets stay in registers: gate * post and pre.
// PER_ROW: the gate is a row's own (token or full form) and joins post in the row.
template <typename T, typename W, int VEC, int NV, bool PER_ROW, bool LED, typename R>
__device__ __forceinline__ void norm_forward_rows(const NormParams& p, char* smem, R& ring, const Columns c) {
  const bool full = PER_ROW && p.gate_form == TNX_GATE_FULL;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  float pg[NV][VEC];
  elem::Pack<W, VEC> pre[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int col = c.first + n * c.step;
    if (col < c.limit) {
      column_load<W, VEC, LED>(static_cast<const W*>(p.post) + col, pg[n]);
      pre[n] = column_pack<W, VEC, LED>(static_cast<const W*>(p.pre) + col);
      if (!PER_ROW && p.gate_form == TNX_GATE_CHANNEL) {
        float g[VEC];
        column_load<W, VEC, LED>(static_cast<const W*>(p.gate) + col, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) pg[n][j] *= g[j];
      }
    }
  }
  int levels = 0;
  while ((32 << levels) < static_cast<int>(blockDim.x)) ++levels;
  bool ok = true;
  // (rows <= 2^30: row numbers cannot overflow)
  for (; ring.row < p.rows; ring.next()) {
    const long long row = ring.row;
    float token = 1.f;
    if (PER_ROW && !full) token = elem::to_float(static_cast<const W*>(p.gate)[row * p.ld_gate]);
    ok = ring.wait(p.timeout_ns);
    const T* y_row = reinterpret_cast<const T*>(smem + kCtrlBytes + ring.at(0));
    const T* r_row = reinterpret_cast<const T*>(smem + kCtrlBytes + ring.at(1));
    const W* g_row = reinterpret_cast<const W*>(smem + kCtrlBytes + (full ? ring.at(2) : 0u));
    elem::Pack<T, VEC> y[NV];
    float h[NV][VEC];  // gate * post, then h
    float ss[1] = {0.f};
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int col = c.first + n * c.step;
      if (col < c.limit) {
        y[n] = *reinterpret_cast<const elem::Pack<T, VEC>*>(y_row + col);
#pragma unroll
        for (int j = 0; j < VEC; ++j) ss[0] += elem::to_float(y[n].v[j]) * elem::to_float(y[n].v[j]);
      }
    }
    block_sum(ss, ring.ctrl->sums[0], levels, ok);
    if (!ok) break;
    const float r1 = rsqrtf(ss[0] * inv_cols + p.eps);
    ss[0] = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int col = c.first + n * c.step;
      if (col < c.limit) {
        float r[VEC], g[VEC];
        elem::load<T, VEC>(r_row + col, r);
        if (full) elem::load<W, VEC>(g_row + col, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float b = elem::to_float(y[n].v[j]) * r1 * pg[n][j];
          h[n][j] = p.alpha * r[j] + (!PER_ROW ? b : full ? g[j] * b : token * b);
          ss[0] += h[n][j] * h[n][j];
        }
      }
    }
    block_sum(ss, ring.ctrl->sums[1], levels, ok);
    const float r2 = rsqrtf(ss[0] * inv_cols + p.eps);
    ring.refill();
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int col = c.first + n * c.step;
      if (col < c.limit) {
        float out[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = h[n][j] * r2 * elem::to_float(pre[n].v[j]);
        elem::store<T, VEC>(static_cast<T*>(p.h) + row * p.cols + col, h[n]);
        elem::store<T, VEC>(static_cast<T*>(p.n) + row * p.cols + col, out);
      }
    }
    if (p.stats != nullptr && threadIdx.x == 0) *reinterpret_cast<float2*>(p.stats + 2 * row) = make_float2(r1, r2);
  }
  if (!ok) ring.give_up(p.status);
}
template <typename T, typename W, int VEC, int NV, bool PER_ROW, bool LED, typename R>
__device__ __forceinline__ void norm_backward_rows(const NormParams& p, char* smem, R& ring, const Columns c) {
  const bool full = PER_ROW && p.gate_form == TNX_GATE_FULL;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  float s_a[NV][VEC], s_pre[NV][VEC];  // column sums: dh' a (times the row's gate), dn h r2
  float pg[NV][VEC];
  elem::Pack<W, VEC> pre[NV];
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int col = c.first + n * c.step;
#pragma unroll
    for (int j = 0; j < VEC; ++j) s_a[n][j] = s_pre[n][j] = 0.f;
    if (col < c.limit) {
      column_load<W, VEC, LED>(static_cast<const W*>(p.post) + col, pg[n]);
      pre[n] = column_pack<W, VEC, LED>(static_cast<const W*>(p.pre) + col);
      if (!PER_ROW && p.gate_form == TNX_GATE_CHANNEL) {
        float g[VEC];
        column_load<W, VEC, LED>(static_cast<const W*>(p.gate) + col, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) pg[n][j] *= g[j];
      }
    }
  }
  int levels = 0;
  while ((32 << levels) < static_cast<int>(blockDim.x)) ++levels;
  bool ok = true;
  // (rows <= 2^30: row numbers cannot overflow)
  for (; ring.row < p.rows; ring.next()) {
    const long long row = ring.row;
    const float2 norms = *reinterpret_cast<const float2*>(p.stats + 2 * row);
    const float r1 = norms.x, r2 = norms.y;
    float token = 1.f;
    if (PER_ROW && !full) token = elem::to_float(static_cast<const W*>(p.gate)[row * p.ld_gate]);
    ok = ring.wait(p.timeout_ns);
    const T* y_row = reinterpret_cast<const T*>(smem + kCtrlBytes + ring.at(0));
    const T* r_row = reinterpret_cast<const T*>(smem + kCtrlBytes + ring.at(1));
    const T* dh_row = reinterpret_cast<const T*>(smem + kCtrlBytes + ring.at(2));
    const T* dn_row = reinterpret_cast<const T*>(smem + kCtrlBytes + ring.at(3));
    const W* g_row = reinterpret_cast<const W*>(smem + kCtrlBytes + (full ? ring.at(4) : 0u));
    float h[NV][VEC];
    elem::Pack<T, VEC> y[NV];
    float s_uh[1] = {0.f};
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int col = c.first + n * c.step;
      if (col < c.limit) {
        float g[VEC], u[VEC];
        y[n] = *reinterpret_cast<const elem::Pack<T, VEC>*>(y_row + col);
        elem::load<T, VEC>(r_row + col, h[n]);
        elem::load<T, VEC>(dn_row + col, u);
        if (full) elem::load<W, VEC>(g_row + col, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float b = elem::to_float(y[n].v[j]) * r1 * pg[n][j];
          h[n][j] = p.alpha * h[n][j] + (!PER_ROW ? b : full ? g[j] * b : token * b);
          s_pre[n][j] += u[j] * (h[n][j] * r2);
          s_uh[0] += u[j] * elem::to_float(pre[n].v[j]) * h[n][j];
        }
      }
    }
    block_sum(s_uh, ring.ctrl->sums[0], levels, ok);
    if (!ok) break;
    const float k = s_uh[0] * inv_cols * r2 * r2;
    float s_va = 0.f, s_g = 0.f;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int col = c.first + n * c.step;
      if (col < c.limit) {
        float g[VEC], u[VEC], d[VEC], dg[VEC];
        elem::load<T, VEC>(dh_row + col, d);
        elem::load<T, VEC>(dn_row + col, u);
        if (full) elem::load<W, VEC>(g_row + col, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float a = elem::to_float(y[n].v[j]) * r1;
          const float dh = d[j] + r2 * (u[j] * elem::to_float(pre[n].v[j]) - h[n][j] * k);
          const float gate = !PER_ROW ? 1.f : full ? g[j] : token;
          d[j] = p.alpha * dh;
          s_a[n][j] += gate * dh * a;
          if (PER_ROW) {
            dg[j] = dh * (a * pg[n][j]);
            s_g += dg[j];
          }
          h[n][j] = gate * dh * pg[n][j];  // (v from here on)
          s_va += h[n][j] * a;
        }
        elem::store<T, VEC>(static_cast<T*>(p.dres) + row * p.cols + col, d);
        if (full) elem::store<W, VEC>(static_cast<W*>(p.dgate) + row * p.cols + col, dg);
      }
    }
    float both[PER_ROW ? 2 : 1] = {s_va};
    if (PER_ROW) both[PER_ROW ? 1 : 0] = s_g;
    block_sum(both, ring.ctrl->sums[1], levels, ok);
    ring.refill();
    const float m = both[0] * inv_cols;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int col = c.first + n * c.step;
      if (col < c.limit) {
        float out[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) out[j] = r1 * (h[n][j] - elem::to_float(y[n].v[j]) * r1 * m);
        elem::store<T, VEC>(static_cast<T*>(p.dy) + row * p.cols + col, out);
      }
    }
    if (PER_ROW && !full && threadIdx.x == 0) static_cast<W*>(p.dgate)[row] = elem::from_float<W>(both[PER_ROW ? 1 : 0]);
  }
  if (!ok) ring.give_up(p.status);
  float* mine = p.partial + static_cast<long long>(blockIdx.x) * p.sums * p.cols;
#pragma unroll
  for (int n = 0; n < NV; ++n) {
    const int col = c.first + n * c.step;
    if (col < c.limit) {
      if (!PER_ROW && p.gate_form == TNX_GATE_CHANNEL) {
        float g[VEC], post[VEC];
        column_load<W, VEC, LED>(static_cast<const W*>(p.gate) + col, g);
        column_load<W, VEC, LED>(static_cast<const W*>(p.post) + col, post);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          post[j] *= s_a[n][j];
          s_a[n][j] *= g[j];
        }
        column_store<VEC, LED>(mine + 2 * static_cast<long long>(p.cols) + col, post);
      }
      column_store<VEC, LED>(mine + col, s_a[n]);
      column_store<VEC, LED>(mine + p.cols + col, s_pre[n]);
    }
  }
}
template <typename T, typename W, int VEC, int NV, bool PER_ROW, bool LED>
__global__ void __launch_bounds__(ring_threads(VEC, NV, LED), ring_blocks(VEC, NV, LED, false)) norm_forward_ring_kernel(const NormParams p) {
  extern __shared__ __align__(128) char smem[];
  Ring<VEC == 1 || LED> ring(smem, p);
  ring.template add<T>(p.y, p.ld_y, p.cols);
  ring.template add<T>(p.res, p.ld_res, p.cols);
  if (PER_ROW && p.gate_form == TNX_GATE_FULL) ring.template add<W>(p.gate, p.ld_gate, p.cols);
  ring.start();
  if constexpr (LED) {
    const Led led(p.cols, VEC);
    if (led.edge)
      norm_forward_rows<T, W, 1, 1, PER_ROW, false>(p, smem, ring, led.edges(p.cols));
    else
      norm_forward_rows<T, W, VEC, NV, PER_ROW, true>(p, smem, ring, led.vectors(p.cols, VEC));
  } else {
    norm_forward_rows<T, W, VEC, NV, PER_ROW, false>(
        p, smem, ring, {static_cast<int>(threadIdx.x) * VEC, static_cast<int>(blockDim.x) * VEC, p.cols});
  }
}

// The sums of norm_backward_kernel.  A gate per channel leaves the sum over rows, so that one sum
// S = sum of dh' a gives both dpost = gate S and dgate = post S.
template <typename T, typename W, int VEC, int NV, bool PER_ROW, bool LED>
__global__ void __launch_bounds__(ring_threads(VEC, NV, LED), ring_blocks(VEC, NV, LED, true)) norm_backward_ring_kernel(const NormParams p) {
  extern __shared__ __align__(128) char smem[];
  Ring<VEC == 1 || LED> ring(smem, p);
  ring.template add<T>(p.y, p.ld_y, p.cols);
  ring.template add<T>(p.res, p.ld_res, p.cols);
  ring.template add<T>(p.dh, p.ld_dh, p.cols);
  ring.template add<T>(p.dn, p.ld_dn, p.cols);
  if (PER_ROW && p.gate_form == TNX_GATE_FULL) ring.template add<W>(p.gate, p.ld_gate, p.cols);
  ring.start();
  if constexpr (LED) {
    const Led led(p.cols, VEC);
    if (led.edge)
      norm_backward_rows<T, W, 1, 1, PER_ROW, false>(p, smem, ring, led.edges(p.cols));
    else
      norm_backward_rows<T, W, VEC, NV, PER_ROW, true>(p, smem, ring, led.vectors(p.cols, VEC));
  } else {
    norm_backward_rows<T, W, VEC, NV, PER_ROW, false>(
        p, smem, ring, {static_cast<int>(threadIdx.x) * VEC, static_cast<int>(blockDim.x) * VEC, p.cols});
  }
}

// out[s][c] = sum over blocks b of partial[b][s][c], b in a fixed order: 32 columns x 32 strands
// of blocks per thread block, the strands added pairwise.
template <typename W>
__global__ void __launch_bounds__(1024) norm_column_sums(const float* partial, int blocks, int sums, int cols,
                                                         W* post, W* pre, W* gate) {
  __shared__ float acc[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  const int s = blockIdx.y;
  float v = 0.f;
  if (col < cols)
    for (int b = threadIdx.y; b < blocks; b += 32)
      v += partial[(static_cast<long long>(b) * sums + s) * cols + col];
  acc[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = acc[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int out_col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && out_col < cols) {
    W* out = s == 0 ? post : s == 1 ? pre : gate;
    out[out_col] = elem::from_float<W>(v);
  }
}

inline int cdiv(int a, int b) { return (a + b - 1) / b; }

// Vector width, vectors per thread, threads and rows of a block for one call; depth > 0: a ring
// kernel with that many rows in flight and `smem` bytes per block.
// led: rows do not start on 16-byte boundaries, but in all tensors alike.
struct NormShape {
  int vec, nv, threads, rows, depth, smem, blocks;
  int period;  // blocks that walk rows are a multiple of this
  bool led;
};

// A row's threads: one vector each while a block holds the row, then two, four, ... each.
// How the rows lie.
enum Rows {
  kAligned,  // all start on 16-byte boundaries
  kAlike,    // all tensors do, and row r of each starts r * cols elements (to a whole vector) after that
  kAnyhow,
  kRepeated  // anyhow, and a tensor's rows overlap: a copy to the next boundary could pass its end
};
void pick_shape(const tnx_norm_problem& p, Rows how, bool backward, NormShape* s) {
  const int wide = p.dtype == TNX_F32 ? 4 : 8;
  const bool aligned = how == kAligned;
  // Rows in flight: what fits a third (forward) or half (backward) of an SM's shared memory, four
  // at most; and enough rows that a block has several.
  const int size = p.dtype == TNX_F32 ? 4 : 2, wsize = p.weight_dtype == TNX_F32 ? 4 : 2;
  const int slot = (backward ? 4 : 2) * static_cast<int>(ring_row_bytes(p.cols, size)) +
                   (p.gate_form == TNX_GATE_FULL ? static_cast<int>(ring_row_bytes(p.cols, wsize)) : 0);
  const int share = kMaxDynamicSmem / (backward ? 2 : 3) - 1024;
  s->depth = 0;
  if (p.rows >= 4 * sm_count() && how != kRepeated) {
    s->depth = (share - kCtrlBytes) / slot;
    if (s->depth < 2) s->depth = (kMaxDynamicSmem - kCtrlBytes) / slot;
    if (s->depth > kMaxDepth) s->depth = kMaxDepth;
    if (s->depth < 2) s->depth = 0;
  }
  // Whole vectors against single elements, fp32 weights and a channel gate, us forward/backward:
  // 4000 x 7001 bf16 59/115 against 119/342, 32768 x 301 bf16 41/82 against 86/131; 50000 x 67 fp32
  // 35/64 against 37/61, no gain: rows that short are a few warps either way.  (The longest rows do
  // not fit 480 threads.)
  const int longest = 480 * (wide == 8 ? 4 : 8) * wide;
  s->led = how == kAlike && s->depth > 0 && p.cols >= 16 * wide && p.cols <= longest;
  s->vec = aligned || s->led ? wide : 1;
  const int vectors = s->led ? p.cols / wide : cdiv(p.cols, s->vec);
  s->nv = 1;
  while (cdiv(vectors, s->nv) > max_threads(s->vec, s->nv, s->led)) s->nv *= 2;
  s->threads = cdiv(cdiv(vectors, s->nv), 32) * 32;
  if (s->led) s->threads += 32;
  s->rows = backward || s->depth > 0 ? 1 : s->threads >= 256 ? 1 : 256 / s->threads;
  s->smem = s->depth > 0 ? kCtrlBytes + s->depth * slot : 0;
  // Blocks that walk rows: as many as can be resident (resident_blocks has the last word), never more
  // than there are rows.
  int per_sm = 2;
  if (s->depth > 0) {
    const int by_smem = (kMaxDynamicSmem + 1024) / (s->smem + 1024), by_regs = (backward ? 768 : 1024) / s->threads;
    per_sm = by_smem < by_regs ? by_smem : by_regs;
    if (per_sm < 1) per_sm = 1;
    if (per_sm > 16) per_sm = 16;
  }
  s->blocks = p.rows < per_sm * sm_count() ? p.rows : per_sm * sm_count();
  s->period = 1;
  if (s->depth > 0 && !aligned) {
    int period = wide;  // rows after which all tensors are as far behind a boundary again
    while (s->led && period > 1 && period / 2 * static_cast<long long>(p.cols) % wide == 0) period /= 2;
    s->period = period;
    s->blocks -= s->blocks % period;  // (there are at least four rows per SM)
  }
}

int norm_check(const tnx_norm_problem* p, bool backward, const void* const* ptrs, int count,
               const long long* pitches, int pitch_count, NormShape* s) {
  if (p == nullptr) {
    set_error("problem is NULL");
    return TNX_ERR_INVALID;
  }
  if (p->rows < 0 || p->rows > (1 << 30) || p->cols < 1 || p->cols > kMaxCols) {
    set_error("the norm needs 0 to 2^30 rows and 1 <= cols <= %d (got %d x %d)", kMaxCols, p->rows, p->cols);
    return TNX_ERR_INVALID;
  }
  if (p->dtype < TNX_F16 || p->dtype > TNX_F32 || (p->weight_dtype != p->dtype && p->weight_dtype != TNX_F32)) {
    set_error("weight_dtype must be the dtype or TNX_F32 (got dtype %d, weight_dtype %d)", p->dtype, p->weight_dtype);
    return TNX_ERR_INVALID;
  }
  if (p->gate_form < TNX_GATE_NONE || p->gate_form > TNX_GATE_FULL) {
    set_error("unknown gate form %d", p->gate_form);
    return TNX_ERR_INVALID;
  }
  if (!(p->eps > 0.f)) {
    set_error("eps must be positive");
    return TNX_ERR_INVALID;
  }
  const int wide = p->dtype == TNX_F32 ? 4 : 8;
  bool based = true, aligned = p->cols % wide == 0, alike = true, apart = true;
  for (int i = 0; i < count; ++i) based = based && (reinterpret_cast<uintptr_t>(ptrs[i]) & 15u) == 0;
  for (int i = 0; i < pitch_count; ++i) {
    if (pitches[i] < 0) {
      set_error("negative row pitches are not supported");
      return TNX_ERR_INVALID;
    }
    aligned = aligned && pitches[i] % wide == 0;
    alike = alike && pitches[i] % wide == p->cols % wide;
    apart = apart && pitches[i] >= p->cols;
  }
  pick_shape(*p, based && aligned ? kAligned : !apart ? kRepeated : based && alike ? kAlike : kAnyhow, backward, s);
  return TNX_OK;
}

using NormFn = void (*)(const NormParams);

// A kernel: plain, or a ring kernel with a gate per row or not.
struct Pick {
  bool ring, per_row, led, backward;
};
template <typename T, typename W, int VEC, int NV, bool LED>
NormFn pick_ring(const Pick& k) {
  if (k.per_row)
    return k.backward ? norm_backward_ring_kernel<T, W, VEC, NV, true, LED> : norm_forward_ring_kernel<T, W, VEC, NV, true, LED>;
  return k.backward ? norm_backward_ring_kernel<T, W, VEC, NV, false, LED> : norm_forward_ring_kernel<T, W, VEC, NV, false, LED>;
}
template <typename T, typename W, int VEC, int NV>
NormFn pick_form(const Pick& k) {
  if (!k.ring) return k.backward ? norm_backward_kernel<T, W, VEC, NV> : norm_forward_kernel<T, W, VEC, NV>;
  if constexpr (VEC > 1)
    if (k.led) return pick_ring<T, W, VEC, NV, true>(k);
  return pick_ring<T, W, VEC, NV, false>(k);
}
template <typename T, typename W, int VEC>
NormFn pick_nv(int nv, const Pick& k) {
  if (nv == 1) return pick_form<T, W, VEC, 1>(k);
  if (nv == 2) return pick_form<T, W, VEC, 2>(k);
  if (nv == 4) return pick_form<T, W, VEC, 4>(k);
  // (16384 columns: four vectors of eight, eight of four or 32 single elements)
  if constexpr (VEC != 8)
    if (nv == 8) return pick_form<T, W, VEC, 8>(k);
  if constexpr (VEC == 1) {
    if (nv == 16) return pick_form<T, W, VEC, 16>(k);
    if (nv == 32) return pick_form<T, W, VEC, 32>(k);
  }
  return nullptr;
}
template <typename T, typename W, int WIDE>
NormFn pick_vec(const NormShape& s, const Pick& k) {
  return s.vec == 1 ? pick_nv<T, W, 1>(s.nv, k) : pick_nv<T, W, WIDE>(s.nv, k);
}
NormFn pick_norm(const tnx_norm_problem& p, const NormShape& s, bool backward) {
  const Pick k = {s.depth > 0, p.gate_form == TNX_GATE_TOKEN || p.gate_form == TNX_GATE_FULL, s.led, backward};
  const bool same = p.weight_dtype == p.dtype;
  if (p.dtype == TNX_F32) return pick_vec<float, float, 4>(s, k);
  if (p.dtype == TNX_F16)
    return same ? pick_vec<__half, __half, 8>(s, k) : pick_vec<__half, float, 8>(s, k);
  return same ? pick_vec<__nv_bfloat16, __nv_bfloat16, 8>(s, k)
              : pick_vec<__nv_bfloat16, float, 8>(s, k);
}

// The column sums of the backward pass at most: those of the form with the most blocks.
int most_blocks(const tnx_norm_problem& p) {
  int most = 0;
  for (const Rows how : {kAligned, kAlike, kAnyhow, kRepeated}) {
    NormShape s;
    pick_shape(p, how, true, &s);
    if (s.blocks > most) most = s.blocks;
  }
  return most;
}

// Opts a ring kernel into its dynamic shared memory, once per (kernel, device).
int allow_smem(NormFn fn, int bytes) {
  if (bytes <= 48 * 1024) return TNX_OK;
  constexpr int kSlots = 64;
  static std::mutex mu;
  static NormFn fns[kSlots];
  static int devs[kSlots], used = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) {
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < used; ++i)
      if (fns[i] == fn && devs[i] == dev) return TNX_OK;
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                             kMaxDynamicSmem);
    if (e == cudaSuccess && used < kSlots) {
      fns[used] = fn;
      devs[used++] = dev;
    }
  }
  if (e == cudaSuccess) return TNX_OK;
  set_error("gated residual norm: shared memory: %s", cudaGetErrorString(e));
  (void)cudaGetLastError();
  return TNX_ERR_CUDA;
}

// The blocks of a ring kernel that are resident together: one that started only after another had
// finished would double the time.
int resident_blocks(NormFn fn, const NormShape& s) {
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, reinterpret_cast<const void*>(fn), s.threads, s.smem) != cudaSuccess)
    (void)cudaGetLastError();
  if (per_sm < 1 || per_sm * sm_count() >= s.blocks) return s.blocks;
  const int blocks = per_sm * sm_count();
  return blocks - blocks % s.period;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TNX_OK;
  set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
  return TNX_ERR_CUDA;
}

// edge_rows() of the tensor with the most, all of them at least as wide as the rows are long.
int most_edge_rows(const tnx_norm_problem& p, const long long* pitches, int count) {
  long long least = pitches[0];
  for (int k = 1; k < count; ++k) least = pitches[k] < least ? pitches[k] : least;
  return edge_rows(least * (p.dtype == TNX_F32 ? 4 : 2));  // (a gate of fp32 has fewer)
}

// Bytes that the bulk copies of a tensor's rows read before its first or past its last byte, at most.
int64_t outside(const void* base, int64_t rows, int64_t pitch, uint32_t row_bytes, int edge, bool moved) {
  const int64_t start = static_cast<int64_t>(reinterpret_cast<uintptr_t>(base)), end = start + (rows - 1) * pitch + row_bytes;
  int64_t most = 0;
  for (int64_t r = 0; r < rows; ++r) {
    const int64_t at = start + r * pitch, shift = moved ? at & 15 : 0;
    const CopyPart part = copy_part(static_cast<uint32_t>(shift), row_bytes, moved && r < edge, moved && r >= rows - edge);
    if (part.to == part.from) continue;
    if (start - (at - shift + part.from) > most) most = start - (at - shift + part.from);
    if (at - shift + part.to - end > most) most = at - shift + part.to - end;
  }
  return most;
}

}  // namespace
}  // namespace tnx

extern "C" {

int64_t tnx_selftest_norm_copies(const tnx_norm_problem* problem, const void* y, const void* residual,
                                 const void* gate) {
  using namespace tnx;
  const void* ptrs[] = {y, residual, gate};
  const bool full = problem != nullptr && problem->gate_form == TNX_GATE_FULL;
  NormShape s;
  long long pitches[3] = {};
  if (problem != nullptr) {
    pitches[0] = problem->stride_y;
    pitches[1] = problem->stride_residual;
    pitches[2] = problem->stride_gate;
  }
  const int sources = full ? 3 : 2;
  if (norm_check(problem, false, ptrs, sources, pitches, sources, &s) != TNX_OK) return -2;
  if (s.depth == 0) return -1;
  const int edge = most_edge_rows(*problem, pitches, sources);
  int64_t most = 0;
  for (int k = 0; k < sources; ++k) {
    const int size = (k == 2 ? problem->weight_dtype : problem->dtype) == TNX_F32 ? 4 : 2;
    const int64_t here = outside(ptrs[k], problem->rows, pitches[k] * size, static_cast<uint32_t>(problem->cols * size),
                                 edge, s.vec == 1 || s.led);
    if (here > most) most = here;
  }
  return most;
}

int64_t tnx_gated_residual_norm_workspace(const tnx_norm_problem* problem) {
  if (problem == nullptr || problem->rows <= 0 || problem->cols <= 0) return 0;
  const int sums = problem->gate_form == TNX_GATE_CHANNEL ? 3 : 2;
  return static_cast<int64_t>(tnx::most_blocks(*problem)) * sums * problem->cols * 4;
}

int tnx_gated_residual_norm(const tnx_norm_problem* problem, const void* y, const void* residual,
                            const void* post_weight, const void* pre_weight, const void* gate, void* h, void* n,
                            float* stats, int32_t* status_word, void* stream) {
  using namespace tnx;
  const void* ptrs[] = {y, residual, post_weight, pre_weight, h, n, gate};
  NormShape s;
  long long pitches[3] = {};
  if (problem != nullptr) {
    pitches[0] = problem->stride_y;
    pitches[1] = problem->stride_residual;
    pitches[2] = problem->gate_form == TNX_GATE_FULL ? problem->stride_gate : problem->cols;
  }
  int rc = norm_check(problem, false, ptrs, problem != nullptr && problem->gate_form == TNX_GATE_TOKEN ? 6 : 7,
                      pitches, 3, &s);
  if (rc != TNX_OK) return rc;
  if (problem->rows == 0) return TNX_OK;
  if (y == nullptr || residual == nullptr || post_weight == nullptr || pre_weight == nullptr || h == nullptr ||
      n == nullptr || (problem->gate_form != TNX_GATE_NONE && gate == nullptr)) {
    set_error("NULL operand pointer");
    return TNX_ERR_INVALID;
  }
  NormParams p = {};
  p.rows = problem->rows;
  p.cols = problem->cols;
  p.gate_form = problem->gate_form;
  p.alpha = problem->residual_scale;
  p.eps = problem->eps;
  p.ld_y = problem->stride_y;
  p.ld_res = problem->stride_residual;
  p.ld_gate = problem->stride_gate;
  p.y = y;
  p.res = residual;
  p.post = post_weight;
  p.pre = pre_weight;
  p.gate = gate;
  p.h = h;
  p.n = n;
  p.stats = stats;
  NormFn fn = pick_norm(*problem, s, false);
  if (fn == nullptr) {
    set_error("norm kernel not built for this row length");
    return TNX_ERR_NOT_BUILT;
  }
  p.depth = s.depth;
  if (s.depth > 0) p.edge = most_edge_rows(*problem, pitches, 3);
  p.inner = p.rows - 2 * p.edge;
  p.status = status_word;
  p.timeout_ns = bounded_wait_limit_ns();
  rc = allow_smem(fn, s.smem);
  if (rc != TNX_OK) return rc;
  fn<<<s.depth > 0 ? resident_blocks(fn, s) : cdiv(p.rows, s.rows), dim3(s.threads, s.rows), s.smem, static_cast<cudaStream_t>(stream)>>>(p);
  return launched("gated residual norm");
}

int tnx_gated_residual_norm_backward(const tnx_norm_problem* problem, const void* dh, int64_t stride_dh,
                                     const void* dn, int64_t stride_dn, const void* y, const void* residual,
                                     const void* post_weight, const void* pre_weight, const void* gate,
                                     const float* stats, void* dy, void* dresidual, void* dpost, void* dpre,
                                     void* dgate, void* workspace, size_t workspace_bytes, int32_t* status_word,
                                     void* stream) {
  using namespace tnx;
  const void* ptrs[] = {dh, dn, y, residual, post_weight, pre_weight, dy, dresidual, gate, dgate};
  NormShape s;
  long long pitches[5] = {stride_dh, stride_dn, 0, 0, 0};
  if (problem != nullptr) {
    pitches[2] = problem->stride_y;
    pitches[3] = problem->stride_residual;
    pitches[4] = problem->gate_form == TNX_GATE_FULL ? problem->stride_gate : problem->cols;
  }
  int rc = norm_check(problem, true, ptrs, problem != nullptr && problem->gate_form == TNX_GATE_TOKEN ? 8 : 10,
                      pitches, 5, &s);
  if (rc != TNX_OK) return rc;
  if (dpost == nullptr || dpre == nullptr || (problem->gate_form != TNX_GATE_NONE && dgate == nullptr)) {
    set_error("NULL gradient pointer");
    return TNX_ERR_INVALID;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int blocks = s.blocks;
  if (blocks > 0) {
    if (dh == nullptr || dn == nullptr || y == nullptr || residual == nullptr || post_weight == nullptr ||
        pre_weight == nullptr || stats == nullptr || dy == nullptr || dresidual == nullptr ||
        (problem->gate_form != TNX_GATE_NONE && gate == nullptr)) {
      set_error("NULL operand pointer");
      return TNX_ERR_INVALID;
    }
    const int64_t need = tnx_gated_residual_norm_workspace(problem);
    if (workspace == nullptr || workspace_bytes < static_cast<size_t>(need) ||
        (reinterpret_cast<uintptr_t>(workspace) & 15u)) {
      set_error("the norm's backward pass needs a 16-byte aligned workspace of %lld bytes",
                static_cast<long long>(need));
      return TNX_ERR_INVALID;
    }
  }
  NormParams p = {};
  p.rows = problem->rows;
  p.cols = problem->cols;
  p.gate_form = problem->gate_form;
  p.alpha = problem->residual_scale;
  p.eps = problem->eps;
  p.ld_y = problem->stride_y;
  p.ld_res = problem->stride_residual;
  p.ld_gate = problem->stride_gate;
  p.ld_dh = stride_dh;
  p.ld_dn = stride_dn;
  p.y = y;
  p.res = residual;
  p.post = post_weight;
  p.pre = pre_weight;
  p.gate = gate;
  p.stats = const_cast<float*>(stats);
  p.dh = dh;
  p.dn = dn;
  p.dy = dy;
  p.dres = dresidual;
  p.dgate = dgate;
  p.partial = static_cast<float*>(workspace);
  p.sums = p.gate_form == TNX_GATE_CHANNEL ? 3 : 2;
  if (blocks > 0) {
    NormFn fn = pick_norm(*problem, s, true);
    if (fn == nullptr) {
      set_error("norm kernel not built for this row length");
      return TNX_ERR_NOT_BUILT;
    }
    p.depth = s.depth;
    if (s.depth > 0) p.edge = most_edge_rows(*problem, pitches, 5);
    p.inner = p.rows - 2 * p.edge;
    p.status = status_word;
    p.timeout_ns = bounded_wait_limit_ns();
    rc = allow_smem(fn, s.smem);
    if (rc != TNX_OK) return rc;
    if (s.depth > 0) blocks = resident_blocks(fn, s);
    fn<<<blocks, s.threads, s.smem, st>>>(p);
    rc = launched("gated residual norm, backward");
    if (rc != TNX_OK) return rc;
  }
  const dim3 grid(cdiv(p.cols, 32), p.sums);
  if (problem->weight_dtype == TNX_F32)
    norm_column_sums<float><<<grid, dim3(32, 32), 0, st>>>(p.partial, blocks, p.sums, p.cols,
                                                           static_cast<float*>(dpost), static_cast<float*>(dpre),
                                                           static_cast<float*>(dgate));
  else if (problem->weight_dtype == TNX_F16)
    norm_column_sums<__half><<<grid, dim3(32, 32), 0, st>>>(p.partial, blocks, p.sums, p.cols,
                                                            static_cast<__half*>(dpost), static_cast<__half*>(dpre),
                                                            static_cast<__half*>(dgate));
  else
    norm_column_sums<__nv_bfloat16><<<grid, dim3(32, 32), 0, st>>>(
        p.partial, blocks, p.sums, p.cols, static_cast<__nv_bfloat16*>(dpost), static_cast<__nv_bfloat16*>(dpre),
        static_cast<__nv_bfloat16*>(dgate));
  return launched("gated residual norm, column sums");
}

}  // extern "C"
