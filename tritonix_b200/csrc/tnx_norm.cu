// The seam between two transformer blocks in one pass over the rows:
//     h = residual_scale * residual + gate * rms(y) * post_weight      (the new residual stream)
//     n = rms(h) * pre_weight                                          (input of the next block)
// with rms(v) = v / sqrt(mean(v^2) + eps), and its backward pass.  y is the output of the block
// that has just finished (an MLP or a mixture of experts).
//
// Both passes are bound by HBM: forward reads y and residual and writes h and n (4 values per
// element), backward reads dh, dn, y, residual and writes dy, dresidual (6 values; h and the
// normalised rows are recomputed in fp32 from the saved reciprocal norms, because a weight
// gradient summed from an h that was rounded to 16 bits would carry that rounding).  A row stays
// in the registers of its threads between its first load and its last store, so nothing is read
// twice; reductions and all arithmetic are fp32.
#include <cuda_runtime.h>

#include "tnx_elem.cuh"
#include "tnx_internal.h"

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
};

constexpr int kMaxCols = 16384;
// Threads of a row at most.  Vectors keep eight times the values in registers, so half as many
// threads leave them twice the registers.
__host__ __device__ constexpr int max_threads(int vec) { return vec == 1 ? 1024 : 512; }

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
__global__ void __launch_bounds__(max_threads(VEC)) norm_forward_kernel(const NormParams p) {
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
__global__ void __launch_bounds__(max_threads(VEC)) norm_backward_kernel(const NormParams p) {
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

// Vector width, threads and rows of a block for one call.
struct NormShape {
  int vec, nv, threads, rows;
};

// A row's threads: one vector each while a block holds the row, then two, four, ... each.
void pick_shape(const tnx_norm_problem& p, bool aligned, bool backward, NormShape* s) {
  const int wide = p.dtype == TNX_F32 ? 4 : 8;
  s->vec = aligned && p.cols % wide == 0 ? wide : 1;
  const int vectors = cdiv(p.cols, s->vec);
  const int most = max_threads(s->vec);
  s->nv = 1;
  while (cdiv(vectors, s->nv) > most) s->nv *= 2;
  s->threads = cdiv(cdiv(vectors, s->nv), 32) * 32;
  s->rows = backward ? 1 : s->threads >= 256 ? 1 : 256 / s->threads;
}

int norm_check(const tnx_norm_problem* p, bool backward, const void* const* ptrs, int count,
               const long long* pitches, int pitch_count, NormShape* s) {
  if (p == nullptr) {
    set_error("problem is NULL");
    return TNX_ERR_INVALID;
  }
  if (p->rows < 0 || p->cols < 1 || p->cols > kMaxCols) {
    set_error("the norm needs rows >= 0 and 1 <= cols <= %d (got %d x %d)", kMaxCols, p->rows, p->cols);
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
  bool aligned = true;
  for (int i = 0; i < count; ++i) aligned = aligned && (reinterpret_cast<uintptr_t>(ptrs[i]) & 15u) == 0;
  for (int i = 0; i < pitch_count; ++i) {
    if (pitches[i] < 0) {
      set_error("negative row pitches are not supported");
      return TNX_ERR_INVALID;
    }
    aligned = aligned && pitches[i] % wide == 0;
  }
  pick_shape(*p, aligned, backward, s);
  return TNX_OK;
}

using NormFn = void (*)(const NormParams);

template <typename T, typename W, int VEC>
NormFn pick_nv(int nv, bool backward) {
  if (nv == 1) return backward ? norm_backward_kernel<T, W, VEC, 1> : norm_forward_kernel<T, W, VEC, 1>;
  if (nv == 2) return backward ? norm_backward_kernel<T, W, VEC, 2> : norm_forward_kernel<T, W, VEC, 2>;
  if (nv == 4) return backward ? norm_backward_kernel<T, W, VEC, 4> : norm_forward_kernel<T, W, VEC, 4>;
  // (16384 columns: four vectors of eight, eight of four or sixteen single elements)
  constexpr int kLong = VEC == 8 ? 4 : 8, kLongest = VEC == 1 ? 16 : kLong;
  if (nv == kLong) return backward ? norm_backward_kernel<T, W, VEC, kLong> : norm_forward_kernel<T, W, VEC, kLong>;
  if (nv == kLongest)
    return backward ? norm_backward_kernel<T, W, VEC, kLongest> : norm_forward_kernel<T, W, VEC, kLongest>;
  return nullptr;
}
template <typename T, typename W, int WIDE>
NormFn pick_vec(const NormShape& s, bool backward) {
  return s.vec == 1 ? pick_nv<T, W, 1>(s.nv, backward) : pick_nv<T, W, WIDE>(s.nv, backward);
}
NormFn pick_norm(const tnx_norm_problem& p, const NormShape& s, bool backward) {
  const bool same = p.weight_dtype == p.dtype;
  if (p.dtype == TNX_F32) return pick_vec<float, float, 4>(s, backward);
  if (p.dtype == TNX_F16)
    return same ? pick_vec<__half, __half, 8>(s, backward) : pick_vec<__half, float, 8>(s, backward);
  return same ? pick_vec<__nv_bfloat16, __nv_bfloat16, 8>(s, backward)
              : pick_vec<__nv_bfloat16, float, 8>(s, backward);
}

// Blocks of the backward pass: two per SM, never more than there are rows.
int backward_blocks(const tnx_norm_problem& p) {
  const int most = 2 * sm_count();
  return p.rows < most ? p.rows : most;
}

int launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TNX_OK;
  set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
  return TNX_ERR_CUDA;
}

}  // namespace
}  // namespace tnx

extern "C" {

int64_t tnx_gated_residual_norm_workspace(const tnx_norm_problem* problem) {
  if (problem == nullptr || problem->rows <= 0 || problem->cols <= 0) return 0;
  const int sums = problem->gate_form == TNX_GATE_CHANNEL ? 3 : 2;
  return static_cast<int64_t>(tnx::backward_blocks(*problem)) * sums * problem->cols * 4;
}

int tnx_gated_residual_norm(const tnx_norm_problem* problem, const void* y, const void* residual,
                            const void* post_weight, const void* pre_weight, const void* gate, void* h, void* n,
                            float* stats, void* stream) {
  using namespace tnx;
  const void* ptrs[] = {y, residual, post_weight, pre_weight, h, n, gate};
  NormShape s;
  long long pitches[3] = {0, 0, 0};
  if (problem != nullptr) {
    pitches[0] = problem->stride_y;
    pitches[1] = problem->stride_residual;
    pitches[2] = problem->gate_form == TNX_GATE_FULL ? problem->stride_gate : 0;
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
  fn<<<cdiv(p.rows, s.rows), dim3(s.threads, s.rows), 0, static_cast<cudaStream_t>(stream)>>>(p);
  return launched("gated residual norm");
}

int tnx_gated_residual_norm_backward(const tnx_norm_problem* problem, const void* dh, int64_t stride_dh,
                                     const void* dn, int64_t stride_dn, const void* y, const void* residual,
                                     const void* post_weight, const void* pre_weight, const void* gate,
                                     const float* stats, void* dy, void* dresidual, void* dpost, void* dpre,
                                     void* dgate, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tnx;
  const void* ptrs[] = {dh, dn, y, residual, post_weight, pre_weight, dy, dresidual, gate, dgate};
  NormShape s;
  long long pitches[5] = {stride_dh, stride_dn, 0, 0, 0};
  if (problem != nullptr) {
    pitches[2] = problem->stride_y;
    pitches[3] = problem->stride_residual;
    pitches[4] = problem->gate_form == TNX_GATE_FULL ? problem->stride_gate : 0;
  }
  int rc = norm_check(problem, true, ptrs, problem != nullptr && problem->gate_form == TNX_GATE_TOKEN ? 8 : 10,
                      pitches, 5, &s);
  if (rc != TNX_OK) return rc;
  if (dpost == nullptr || dpre == nullptr || (problem->gate_form != TNX_GATE_NONE && dgate == nullptr)) {
    set_error("NULL gradient pointer");
    return TNX_ERR_INVALID;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int blocks = backward_blocks(*problem);
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
    fn<<<blocks, s.threads, 0, st>>>(p);
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
