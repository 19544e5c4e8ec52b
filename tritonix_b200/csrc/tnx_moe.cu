// Experts' gated products for sm_100a:
//     y[t] = sum over slots s of  w[t, s] * ( act(x[t].W1[e]) * (x[t].W2[e]) ) . W3[e],  e = ids[t, s]
// with W12 = W1/W2 column-interleaved per expert, and its backward pass.
//
//  * A (token, slot) pair is a row of a grouped problem.  plan_* sorts the pairs by expert (stable:
//    rows of an expert keep the pairs' order, so every sum has a fixed order) and pads each expert
//    to whole row tiles.  Nothing about the routing is needed on the host.
//  * moe_gemm_kernel runs the products on the TMA -> shared memory -> tcgen05 -> TMEM pipeline of
//    the library's GEMM, with X and dY the rows of x and dy in expert order:
//        kGateUp  H = w * act(X W1) * (X W2)          weights N-major
//        kDown    O = H W3                            fp32, one row per pair
//        kDHidden dH = dY W3^T, then dGU and dw       weights K-major
//        kDX      O = dGU W12^T                       fp32, one row per pair
//        kDW12, kDW3   X^T dGU and H^T dY per expert  K = the expert's rows
//    permute_kernel copies rows into expert order.  With few rows per expert the copy engine picks
//    them itself instead (kGateUpGather, tile::gather4, one lane per four rows): a gather of four
//    128-byte row pieces was measured to take about as long as a whole box of rows (40-75 cycles),
//    so 128 rows by gathers cost 2.3 times the tensor cores' time (8192 tokens, 64 experts
//    2048/1024: gate/up product 1287 us gathered), while a few rows cost nothing and save a launch.
//    The routing weight is applied to the hidden activation before it is rounded: the rows of O
//    only need adding, and H is the very operand dW3 needs, so no value on the way is rounded
//    twice.
//  * combine_kernel adds a token's rows of O in slot order (fp32) and rounds once.
//  * The gate/up products are kept in fp32 for the backward pass: rounding them to 16 bits would
//    add two more roundings to every gradient.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>
#include <utility>
#include <vector>

#include "tnx_elem.cuh"
#include "tnx_internal.h"
#include "tnx_ptx.cuh"

namespace tnx {

namespace {

constexpr int kMaxExperts = 512;
constexpr int kRows = 128;       // rows per CTA (TMEM lanes)
constexpr int kTileK = 64;       // K elements per ring slot: one 128-byte swizzle row
constexpr int kThreads = 192;    // producer warp, MMA warp, four epilogue warps
constexpr int kEpiThreads = 128;
constexpr int kEpiBarrier = 1;
constexpr int kAtomBytes = 128;
constexpr int kBoxBytes = kRows * kAtomBytes;  // a 128-row box of 128-byte rows
constexpr int kMaxStages = 8;
constexpr int kCtrlBytes = 512;
constexpr int kAlignSlack = 1024;

constexpr int kAbortProducer = 0x301;
constexpr int kAbortMma = 0x302;
constexpr int kAbortEpilogue = 0x303;

enum Mode { kGateUp, kGateUpGather, kDown, kDHidden, kDX, kDW12, kDW3 };

// What a mode's operands look like.
template <int MODE>
struct Traits {
  static constexpr bool wgrad = MODE == kDW12 || MODE == kDW3;
  static constexpr bool gather_a = MODE == kGateUpGather;
  static constexpr bool gate_up = MODE == kGateUp || MODE == kGateUpGather;
  static constexpr bool b_kmajor = MODE == kDHidden || MODE == kDX;
};
// Accumulator columns per tile.  (dHidden streams gate/up through shared memory as well; a
// single CTA then has room for 128 columns only.)
constexpr int tile_n(int mode, int cta_group) { return mode == kDHidden && cta_group == 1 ? 128 : 256; }
constexpr int staging_boxes(int mode) { return mode == kDHidden ? 6 : 2; }

// Where the pairs went (device memory, written by the plan kernels).
struct Plan {
  int* tiles;        // [1] row tiles in use
  int* count;        // [experts] rows of an expert
  int* start;        // [experts] its first (padded) row
  int* tile_expert;  // [max_tiles]
  int* row_token;    // [max_rows] token of a row (rows in use only)
  float* row_weight; // [max_rows]
  int* pos;          // [pairs] row of a pair, -1 where its id is no expert
};

struct GemmParams {
  Plan plan;
  int experts;
  int tile_rows;   // rows per row tile (kRows * CTA_GROUP)
  int num_kb;      // K blocks (not wgrad)
  int cols;        // output columns in accumulator columns
  int tiles_n;     // column tiles
  int band;        // row tiles per band of the tile order
  int tiles_m;     // wgrad: row tiles of the weight
  int m;           // wgrad: rows of the weight
  int activation;
  int save_gu;     // gate/up: also store the fp32 products
  float* part;     // kDown, kDX: O, [max_rows, cols]
  float* dw_part;  // kDHidden: [max_rows, tiles_n]
  int stages;
  int* status;
  unsigned long long timeout_ns;
};

struct Ctrl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint64_t gu_full[2];
  uint32_t tmem_base;
  int abort;
};
static_assert(sizeof(Ctrl) <= kCtrlBytes, "control block too large");

// ------------------------------------------------------------------------------------- plan

// The expert of pair i, -1 where it is none.
__device__ __forceinline__ int pair_expert(const void* ids, int wide, int experts, int i) {
  const long long e = wide ? static_cast<const long long*>(ids)[i] : static_cast<const int*>(ids)[i];
  return e >= 0 && e < experts ? static_cast<int>(e) : -1;
}

struct PlanParams {
  Plan plan;
  const void* ids;
  const float* weights;
  int wide, experts, top_k, pairs, tile_rows;
  int chunk;          // pairs per warp, a multiple of 32
  int chunks;
  int* chunk_counts;  // [chunks][experts] (large problems)
};

// One warp walks its chunk of pairs, 32 at a time, with the ids of eight such steps in flight.
// Pass 1 counts experts in counts[]; pass 2 hands out rows from next[], which holds the chunk's
// first row of every expert.
constexpr int kAhead = 8;
template <typename Step>
__device__ __forceinline__ void walk_chunk(const PlanParams& p, int first, int last, int lane, Step step) {
  for (int base = first; base < last; base += 32 * kAhead) {
    int e[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int i = base + a * 32 + lane;
      e[a] = i < last ? pair_expert(p.ids, p.wide, p.experts, i) : -1;
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      if (base + a * 32 < last) step(base + a * 32 + lane, e[a], __match_any_sync(0xffffffffu, e[a]));
  }
}
__device__ __forceinline__ void count_chunk(const PlanParams& p, int first, int last, int lane, int* counts) {
  walk_chunk(p, first, last, lane, [&](int, int e, unsigned same) {
    if (e >= 0 && lane == __ffs(same) - 1) counts[e] += __popc(same);
    __syncwarp();
  });
}
__device__ __forceinline__ void place_chunk(const PlanParams& p, int first, int last, int lane, int* next) {
  walk_chunk(p, first, last, lane, [&](int i, int e, unsigned same) {
    int row = -1;
    if (e >= 0) row = next[e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) next[e] += __popc(same);
    __syncwarp();
    if (i < last) p.plan.pos[i] = row;
    if (row >= 0) {
      p.plan.row_token[row] = i / p.top_k;
      p.plan.row_weight[row] = p.weights[i];
    }
  });
}

// Given total[e] in shared memory: first row of every expert (in start[]), row tiles and their
// experts.  All threads of the block take part.
__device__ __forceinline__ void lay_out(const PlanParams& p, const int* total, int* start) {
  const int tid = threadIdx.x;
  if (tid < 32) {
    int carry = 0;
    for (int base = 0; base < p.experts; base += 32) {
      const int e = base + tid;
      const int tiles = e < p.experts ? (total[e] + p.tile_rows - 1) / p.tile_rows : 0;
      int sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (tid >= o) sum += v;
      }
      if (e < p.experts) start[e] = (carry + sum - tiles) * p.tile_rows;
      carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (tid == 0) *p.plan.tiles = carry;
  }
  __syncthreads();
  for (int e = tid; e < p.experts; e += blockDim.x) {
    p.plan.count[e] = total[e];
    p.plan.start[e] = start[e];
    const int t0 = start[e] / p.tile_rows, tiles = (total[e] + p.tile_rows - 1) / p.tile_rows;
    for (int i = 0; i < tiles; ++i) p.plan.tile_expert[t0 + i] = e;
  }
}

// Up to kSmallPairs pairs: the whole plan in one block of 32 warps.
constexpr int kSmallPairs = 8192;
constexpr int kSmallWarps = 32;
struct SmallPlanSmem {
  int next[kSmallWarps][kMaxExperts];
  int total[kMaxExperts];
  int start[kMaxExperts];
};
__global__ void __launch_bounds__(kSmallWarps * 32) plan_small_kernel(const PlanParams p) {
  extern __shared__ uint8_t plan_smem[];
  SmallPlanSmem& s = *reinterpret_cast<SmallPlanSmem*>(plan_smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int e = lane; e < p.experts; e += 32) s.next[warp][e] = 0;
  __syncwarp();
  dependency_wait();
  dependency_release();
  const int first = min(warp * p.chunk, p.pairs), last = min(first + p.chunk, p.pairs);
  count_chunk(p, first, last, lane, s.next[warp]);
  __syncthreads();
  for (int e = threadIdx.x; e < p.experts; e += blockDim.x) {
    int run = 0;
#pragma unroll 8
    for (int w = 0; w < kSmallWarps; ++w) {
      const int c = s.next[w][e];
      s.next[w][e] = run;
      run += c;
    }
    s.total[e] = run;
  }
  __syncthreads();
  lay_out(p, s.total, s.start);
  __syncthreads();
  for (int e = lane; e < p.experts; e += 32) s.next[warp][e] += s.start[e];
  __syncwarp();
  place_chunk(p, first, last, lane, s.next[warp]);
}

// More pairs: count per chunk, scan over chunks and experts, place.
constexpr int kChunkWarps = 4;
constexpr int kChunkPairs = 32 * kAhead;
__global__ void __launch_bounds__(kChunkWarps * 32) plan_count_kernel(const PlanParams p) {
  __shared__ int counts[kChunkWarps][kMaxExperts];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunk = blockIdx.x * kChunkWarps + warp;
  for (int e = lane; e < p.experts; e += 32) counts[warp][e] = 0;
  __syncwarp();
  dependency_wait();
  dependency_release();
  if (chunk >= p.chunks) return;
  const int first = chunk * p.chunk, last = min(first + p.chunk, p.pairs);
  count_chunk(p, first, last, lane, counts[warp]);
  for (int e = lane; e < p.experts; e += 32) p.chunk_counts[static_cast<long long>(chunk) * p.experts + e] = counts[warp][e];
}
// Threads (expert, strand): a strand owns a run of chunks, its threads read neighbouring experts.
__global__ void __launch_bounds__(1024) plan_scan_kernel(const PlanParams p) {
  __shared__ int total[kMaxExperts], start[kMaxExperts], strand_sum[1024];
  dependency_wait();
  dependency_release();
  const int strands = 1024 / p.experts;
  const int strand = threadIdx.x / p.experts, e = threadIdx.x - strand * p.experts;
  const int run = (p.chunks + strands - 1) / strands;
  const int c0 = min(strand * run, p.chunks), c1 = strand < strands ? min(c0 + run, p.chunks) : c0;
  int sum = 0;
#pragma unroll 8
  for (int c = c0; c < c1; ++c) sum += p.chunk_counts[static_cast<long long>(c) * p.experts + e];
  strand_sum[threadIdx.x] = sum;
  __syncthreads();
  for (int x = threadIdx.x; x < p.experts; x += blockDim.x) {
    int before = 0;
    for (int t = 0; t < strands; ++t) {
      const int v = strand_sum[t * p.experts + x];
      strand_sum[t * p.experts + x] = before;
      before += v;
    }
    total[x] = before;
  }
  __syncthreads();
  int before = strand_sum[threadIdx.x];
  for (int c = c0; c < c1; c += 8) {
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = c + i < c1 ? p.chunk_counts[static_cast<long long>(c + i) * p.experts + e] : 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c + i < c1) p.chunk_counts[static_cast<long long>(c + i) * p.experts + e] = before;
      before += v[i];
    }
  }
  lay_out(p, total, start);
}
__global__ void __launch_bounds__(kChunkWarps * 32) plan_place_kernel(const PlanParams p) {
  __shared__ int next[kChunkWarps][kMaxExperts];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int chunk = blockIdx.x * kChunkWarps + warp;
  dependency_wait();
  dependency_release();
  if (chunk >= p.chunks) return;
  for (int e = lane; e < p.experts; e += 32)
    next[warp][e] = p.plan.start[e] + p.chunk_counts[static_cast<long long>(chunk) * p.experts + e];
  __syncwarp();
  const int first = chunk * p.chunk, last = min(first + p.chunk, p.pairs);
  place_chunk(p, first, last, lane, next[warp]);
}

// ------------------------------------------------------------------------------------- GEMM

// Gate activation: value and derivative.
__device__ __forceinline__ float2 gate_act(float g, int activation) {
  if (activation == TNX_EPI_GLU_LINEAR) return make_float2(g, 1.f);
  const float s = __fdividef(1.0f, 1.0f + __expf(-g));
  if (activation == TNX_EPI_GLU_SILU) return make_float2(g * s, s * (1.f + g * (1.f - s)));
  return make_float2(s, s * (1.f - s));
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_v4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Four rows of 64 elements each, picked by row number.
template <int CTA_GROUP>
__device__ __forceinline__ void tma_gather4(uint32_t dst, const void* tmap, int x, const int (&rows)[4], uint32_t bar) {
  if (CTA_GROUP == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(rows[0]), "r"(rows[1]), "r"(rows[2]), "r"(rows[3]), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2"
        " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(rows[0]), "r"(rows[1]), "r"(rows[2]), "r"(rows[3]), "r"(bar)
        : "memory");
}
template <int CTA_GROUP>
__device__ __forceinline__ void load_2d(uint32_t dst, const void* tmap, int x, int y, uint32_t bar) {
  if (CTA_GROUP == 1)
    ptx::tma_load_2d(dst, tmap, x, y, bar);
  else
    ptx::tma_load_2d_pair(dst, tmap, x, y, bar);
}
template <int CTA_GROUP>
__device__ __forceinline__ void load_3d(uint32_t dst, const void* tmap, int x, int y, int z, uint32_t bar) {
  if (CTA_GROUP == 1)
    ptx::tma_load_3d(dst, tmap, x, y, z, bar);
  else
    ptx::tma_load_3d_pair(dst, tmap, x, y, z, bar);
}

// One output tile: which expert, where its rows start, how much K there is.
struct Unit {
  int expert;
  int row0;    // first row: padded pair row, or (wgrad) row of the weight
  int valid;   // rows in use from row0 on (may exceed the tile); wgrad: unused
  int col0;    // first accumulator column
  int tile_col;
  int num_kb;
  int k_row0;  // wgrad: first padded pair row of the expert
  int k_rows;  // wgrad: its rows
};

template <int MODE, int TILE_N>
__device__ __forceinline__ Unit decode_unit(const GemmParams& p, int u, int num_tiles) {
  Unit r;
  if (Traits<MODE>::wgrad) {
    // an expert's tiles one after another, column tile by column tile
    const int per = p.tiles_m * p.tiles_n;
    r.expert = u / per;
    const int rem = u - r.expert * per;
    r.tile_col = rem / p.tiles_m;
    r.row0 = (rem - r.tile_col * p.tiles_m) * p.tile_rows;
    r.k_row0 = p.plan.start[r.expert];
    r.k_rows = p.plan.count[r.expert];
    r.num_kb = (r.k_rows + kTileK - 1) / kTileK;
    r.valid = p.m - r.row0;
  } else {
    // bands of `band` row tiles, column tile by column tile inside a band: the CTAs at work share
    // the weight tiles of few experts and the rows of one band through L2
    const int full = p.band * p.tiles_n;
    const int b = u / full;
    const int rem = u - b * full;
    const int rows = min(p.band, num_tiles - b * p.band);
    r.tile_col = rem / rows;
    const int t = b * p.band + (rem - r.tile_col * rows);
    r.expert = p.plan.tile_expert[t];
    r.row0 = t * p.tile_rows;
    r.valid = p.plan.start[r.expert] + p.plan.count[r.expert] - r.row0;
    r.num_kb = p.num_kb;
    r.k_row0 = r.k_rows = 0;
  }
  r.col0 = r.tile_col * TILE_N;
  return r;
}

template <int MODE, int CTA_GROUP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
moe_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                const __grid_constant__ CUtensorMap tmap_c, const __grid_constant__ CUtensorMap tmap_gu,
                const GemmParams p) {
  using T = Traits<MODE>;
  constexpr int TILE_N = tile_n(MODE, CTA_GROUP);
  constexpr int LOAD_N = TILE_N / CTA_GROUP;  // B columns this CTA loads
  constexpr int a_stage_bytes = kRows * kTileK * 2;
  constexpr int b_stage_bytes = LOAD_N * kTileK * 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  const uint32_t base_addr = (raw_addr + 1023u) & ~1023u;
  const uint32_t smem_a = base_addr;
  const uint32_t smem_b = smem_a + p.stages * a_stage_bytes;
  const uint32_t smem_out = smem_b + p.stages * b_stage_bytes;
  const uint32_t smem_gu = smem_out + 2 * kBoxBytes;  // kDHidden: two sets of two boxes
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(smem_raw + (smem_out - raw_addr) + staging_boxes(MODE) * kBoxBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t cta_rank = CTA_GROUP == 2 ? ptx::cluster_ctarank() : 0;
  const bool leader = cta_rank == 0;
  const int cluster_id = blockIdx.x / CTA_GROUP;
  const int num_clusters = gridDim.x / CTA_GROUP;
  volatile int* abort_flag = &ctrl->abort;

  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tmap_a);
    ptx::prefetch_tensormap(&tmap_b);
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->tmem_full[a]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->tmem_empty[a]), 4 * CTA_GROUP);  // one arrive per epilogue warp
      ptx::mbar_init(ptx::smem_u32(&ctrl->gu_full[a]), 1);
    }
    ctrl->abort = 0;
    ptx::fence_mbar_init();
  }
  __syncwarp();
  if (CTA_GROUP == 2) {  // the peer's barriers must exist before anything signals them
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  if (warp == 1) {
    ptx::tmem_alloc<CTA_GROUP>(ptx::smem_u32(&ctrl->tmem_base), 2 * TILE_N);
    ptx::tmem_relinquish<CTA_GROUP>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = ctrl->tmem_base;
  // Everything above touches no global memory and may run under the tail of the kernel before.
  dependency_wait();
  dependency_release();
  const int num_tiles = T::wgrad ? 0 : *p.plan.tiles;
  const int total_units = T::wgrad ? p.experts * p.tiles_m * p.tiles_n : num_tiles * p.tiles_n;

  if (warp == 0) {
    // ===== TMA producer: every lane issues its share of a stage's copies =====
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
      const Unit un = decode_unit<MODE, TILE_N>(p, u, num_tiles);
      const int row0 = un.row0 + static_cast<int>(cta_rank) * kRows;
      const int b_col0 = un.col0 + static_cast<int>(cta_rank) * LOAD_N;
      // Lanes that copy rows of A.  A tile of one CTA with few rows in use fetches only those (the
      // MMA reads the slot's old contents in the other rows, which feed accumulator rows that are
      // never stored); a pair always fetches all.
      int a_lanes = T::gather_a ? 32 : T::wgrad ? 2 : 4;
      if (CTA_GROUP == 1 && !T::wgrad && un.valid < kRows)
        a_lanes = T::gather_a ? (un.valid + 3) / 4 : (un.valid + 31) / 32;
      const uint32_t stage_tx =
          static_cast<uint32_t>(CTA_GROUP * ((T::gather_a ? 512 : T::wgrad ? 8192 : 4096) * a_lanes + b_stage_bytes));
      int rows[4] = {0, 0, 0, 0};
      if (T::gather_a) {
        // rows past the expert's last are copies of that one: addressable, and dropped later
        const int last = un.row0 + un.valid - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) rows[i] = p.plan.row_token[min(row0 + 4 * lane + i, last)];
      }
      for (int kb = 0; kb < un.num_kb; ++kb) {
        const bool got = ptx::mbar_wait(ptx::smem_u32(&ctrl->empty[stage]), phase ^ 1u, abort_flag, p.timeout_ns);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        uint32_t bar = ptx::smem_u32(&ctrl->full[stage]);
        if (leader && lane == 0) ptx::mbar_arrive_expect_tx(bar, stage_tx);
        if (CTA_GROUP == 2) bar = ptx::mapa(bar, 0);  // both CTAs' copies complete on the leader's barrier
        __syncwarp();
        const uint32_t a_dst = smem_a + stage * a_stage_bytes;
        const uint32_t b_dst = smem_b + stage * b_stage_bytes;
        const int k0 = kb * kTileK;
        if (T::wgrad) {
          // K = pair rows; both operands lie in memory as (pair row, column), 64-column atoms
          const int k_row = un.k_row0 + k0;
          if (lane < 2) load_2d<CTA_GROUP>(a_dst + lane * 8192, &tmap_a, row0 + lane * 64, k_row, bar);
          if (lane < LOAD_N / 64) load_2d<CTA_GROUP>(b_dst + lane * 8192, &tmap_b, b_col0 + lane * 64, k_row, bar);
        } else {
          if (T::gather_a) {
            if (lane < a_lanes) tma_gather4<CTA_GROUP>(a_dst + lane * 512, &tmap_a, k0, rows, bar);
          } else if (lane < a_lanes) {
            load_2d<CTA_GROUP>(a_dst + lane * 4096, &tmap_a, k0, row0 + lane * 32, bar);
          }
          if (T::b_kmajor) {
            if (lane == 0) load_3d<CTA_GROUP>(b_dst, &tmap_b, k0, b_col0, un.expert, bar);
          } else if (lane < LOAD_N / 64) {
            load_3d<CTA_GROUP>(b_dst + lane * 8192, &tmap_b, b_col0 + lane * 64, k0, un.expert, bar);
          }
        }
        __syncwarp();
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!ok && lane == 0 && p.status != nullptr) atomicCAS(p.status, 0, kAbortProducer);
  } else if (warp == 1) {
    // ===== MMA issuer (leader CTA) =====
    if (leader && lane == 0) {
      const uint32_t fmt = BF16 ? 1u : 0u;
      const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | ((T::wgrad ? 1u : 0u) << 15) |
                             ((T::b_kmajor ? 0u : 1u) << 16) | (static_cast<uint32_t>(TILE_N >> 3) << 17) |
                             (static_cast<uint32_t>((kRows * CTA_GROUP) >> 4) << 24);
      // K-major operands: rows of 128 bytes, 16 elements of K = 32 bytes further.  MN-major ones:
      // 64-wide atoms of 64 K rows x 128 bytes, 8192 bytes apart, 16 elements of K = 16 rows.
      const uint64_t a_desc = T::wgrad ? ptx::make_smem_desc(0, 8192, 1024) : ptx::make_smem_desc(0, 0, 1024);
      const uint64_t b_desc = T::b_kmajor ? ptx::make_smem_desc(0, 0, 1024) : ptx::make_smem_desc(0, 8192, 1024);
      constexpr uint32_t a_step16 = (T::wgrad ? 2048u : 32u) >> 4;
      constexpr uint32_t b_step16 = (T::b_kmajor ? 32u : 2048u) >> 4;
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
        const int num_kb = T::wgrad ? decode_unit<MODE, TILE_N>(p, u, num_tiles).num_kb : p.num_kb;
        if (num_kb == 0) continue;  // an expert without rows: the epilogue writes zeros by itself
        if (!ptx::mbar_wait<CTA_GROUP == 2>(ptx::smem_u32(&ctrl->tmem_empty[acc]), acc_phase ^ 1u, abort_flag,
                                            p.timeout_ns)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * TILE_N;
        uint32_t accumulate = 0;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!ptx::mbar_wait(ptx::smem_u32(&ctrl->full[stage]), phase, abort_flag, p.timeout_ns)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t a16 = (smem_a + stage * a_stage_bytes) >> 4;
          const uint32_t b16 = (smem_b + stage * b_stage_bytes) >> 4;
#pragma unroll
          for (int k16 = 0; k16 < kTileK / 16; ++k16) {
            ptx::umma_f16<CTA_GROUP>(d_tmem, a_desc | ((a16 + k16 * a_step16) & 0x3fffu),
                                     b_desc | ((b16 + k16 * b_step16) & 0x3fffu), idesc, accumulate);
            accumulate = 1;
          }
          if (CTA_GROUP == 1)
            ptx::umma_commit(ptx::smem_u32(&ctrl->empty[stage]));
          else
            ptx::umma_commit_pair(ptx::smem_u32(&ctrl->empty[stage]), 0x3);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (CTA_GROUP == 1)
          ptx::umma_commit(ptx::smem_u32(&ctrl->tmem_full[acc]));
        else
          ptx::umma_commit_pair(ptx::smem_u32(&ctrl->tmem_full[acc]), 0x3);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok && p.status != nullptr) atomicCAS(p.status, 0, kAbortMma);
    }
  } else {
    // ===== epilogue: warp w owns TMEM lanes 32 (w mod 4) ..., a thread owns a row =====
    const int quarter = warp & 3;
    const int row_in_tile = quarter * 32 + lane;
    const int epi_tid = threadIdx.x - 64;
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t stage_row = static_cast<uint32_t>(row_in_tile) * kAtomBytes;
    const uint32_t sw = static_cast<uint32_t>(row_in_tile & 7);
    int acc = 0;
    uint32_t acc_phase = 0;
    uint32_t stores = 0, gu_chunks = 0;
    bool ok = true;
    // Staging: begin() hands out a box that no store reads any more, end() sends it off.
    auto begin = [&]() -> uint32_t {
      if (epi_tid == 0) ptx::tma_store_wait_read<1>();
      ptx::named_barrier_sync(kEpiBarrier, kEpiThreads);
      return smem_out + (stores & 1u) * kBoxBytes;
    };
    auto end = [&]() {
      ptx::fence_proxy_async_smem();
      ptx::named_barrier_sync(kEpiBarrier, kEpiThreads);
      ++stores;
    };
    for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
      const Unit un = decode_unit<MODE, TILE_N>(p, u, num_tiles);
      const int row0 = un.row0 + static_cast<int>(cta_rank) * kRows;
      const int rows_here = un.valid - static_cast<int>(cta_rank) * kRows;  // rows of this CTA in use (<= 0: none)
      const bool live = row_in_tile < rows_here;

      if (T::wgrad && un.num_kb == 0) {
        // no rows: the gradient is zero
        for (int col = 0; col < TILE_N; col += 64) {
          if (un.col0 + col >= p.cols) break;
          const uint32_t buf = begin();
#pragma unroll
          for (uint32_t piece = 0; piece < 8; ++piece) st_shared_v4(buf + stage_row + piece * 16, 0, 0, 0, 0);
          end();
          if (epi_tid == 0 && row0 < p.m) {
            ptx::tma_store_3d(&tmap_c, un.col0 + col, row0, un.expert, buf);
            ptx::tma_store_commit();
          }
        }
        continue;
      }

      // kDHidden: this tile's gate/up products come in chunks of 32 hidden columns (two boxes of
      // 32 fp32 columns), two chunks ahead.
      const int gu_total = MODE == kDHidden ? (min(TILE_N, p.cols - un.col0) + 31) / 32 : 0;
      auto fetch_gu = [&](int chunk, uint32_t ordinal) {
        const uint32_t set = ordinal & 1u;
        const uint32_t bar = ptx::smem_u32(&ctrl->gu_full[set]);
        const uint32_t dst = smem_gu + set * (2 * kBoxBytes);
        const int x = 2 * (un.col0 + chunk * 32);
        ptx::mbar_arrive_expect_tx(bar, 2 * kBoxBytes);
        ptx::tma_load_2d(dst, &tmap_gu, x, row0, bar);
        ptx::tma_load_2d(dst + kBoxBytes, &tmap_gu, x + 32, row0, bar);
      };
      if (MODE == kDHidden && epi_tid == 0) {
        fetch_gu(0, gu_chunks);
        if (gu_total > 1) fetch_gu(1, gu_chunks + 1);
      }
      const float weight = !T::wgrad && live && (T::gate_up || MODE == kDHidden)
                               ? p.plan.row_weight[row0 + row_in_tile] : 0.f;

      const bool got = ptx::mbar_wait(ptx::smem_u32(&ctrl->tmem_full[acc]), acc_phase, abort_flag, p.timeout_ns);
      if (!ptx::named_barrier_all(kEpiBarrier, kEpiThreads, got)) {
        ok = false;
        break;
      }
      ptx::tc_fence_after_sync();
      const uint32_t t_acc = tmem_base + lane_sel + acc * TILE_N;
      uint32_t r[32];

      if (T::gate_up) {
        if (p.save_gu) {
          for (int col = 0; col < TILE_N; col += 32) {
            if (un.col0 + col >= p.cols) break;
            const uint32_t buf = begin();
            ptx::tmem_ld_32x32(t_acc + col, r);
            ptx::tmem_ld_wait();
#pragma unroll
            for (uint32_t piece = 0; piece < 8; ++piece)
              st_shared_v4(buf + stage_row + (piece ^ sw) * 16, r[piece * 4], r[piece * 4 + 1], r[piece * 4 + 2],
                           r[piece * 4 + 3]);
            end();
            if (epi_tid == 0) {
              ptx::tma_store_2d(&tmap_gu, un.col0 + col, row0, buf);
              ptx::tma_store_commit();
            }
          }
        }
        for (int col = 0; col < TILE_N; col += 128) {
          if (un.col0 + col >= p.cols) break;
          const uint32_t buf = begin();
#pragma unroll
          for (int sub = 0; sub < 4; ++sub) {
            ptx::tmem_ld_32x32(t_acc + col + sub * 32, r);
            ptx::tmem_ld_wait();
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float z0 = weight * gate_act(__uint_as_float(r[4 * j]), p.activation).x * __uint_as_float(r[4 * j + 1]);
              const float z1 = weight * gate_act(__uint_as_float(r[4 * j + 2]), p.activation).x * __uint_as_float(r[4 * j + 3]);
              o[j] = live ? pack2<BF16>(z0, z1) : 0u;
            }
#pragma unroll
            for (uint32_t piece = 0; piece < 2; ++piece)
              st_shared_v4(buf + stage_row + ((sub * 2 + piece) ^ sw) * 16, o[piece * 4], o[piece * 4 + 1],
                           o[piece * 4 + 2], o[piece * 4 + 3]);
          }
          end();
          if (epi_tid == 0) {
            ptx::tma_store_2d(&tmap_c, (un.col0 + col) / 2, row0, buf);
            ptx::tma_store_commit();
          }
        }
      } else if (MODE == kDown || MODE == kDX) {
        if (rows_here <= 32) {
          // few rows: straight from registers, so that unused rows cost no bytes
          if (quarter == 0) {
            float* dst = p.part + static_cast<long long>(row0 + row_in_tile) * p.cols + un.col0;
            for (int col = 0; col < TILE_N; col += 32) {
              if (un.col0 + col >= p.cols) break;
              ptx::tmem_ld_32x32(t_acc + col, r);
              ptx::tmem_ld_wait();
              if (live) {
#pragma unroll
                for (int piece = 0; piece < 8; ++piece)
                  if (un.col0 + col + piece * 4 < p.cols)
                    *reinterpret_cast<float4*>(dst + col + piece * 4) =
                        make_float4(__uint_as_float(r[piece * 4]), __uint_as_float(r[piece * 4 + 1]),
                                    __uint_as_float(r[piece * 4 + 2]), __uint_as_float(r[piece * 4 + 3]));
              }
            }
          }
        } else {
          for (int col = 0; col < TILE_N; col += 32) {
            if (un.col0 + col >= p.cols) break;
            const uint32_t buf = begin();
            ptx::tmem_ld_32x32(t_acc + col, r);
            ptx::tmem_ld_wait();
#pragma unroll
            for (uint32_t piece = 0; piece < 8; ++piece)
              st_shared_v4(buf + stage_row + (piece ^ sw) * 16, r[piece * 4], r[piece * 4 + 1], r[piece * 4 + 2],
                           r[piece * 4 + 3]);
            end();
            if (epi_tid == 0) {
              ptx::tma_store_2d(&tmap_c, un.col0 + col, row0, buf);
              ptx::tma_store_commit();
            }
          }
        }
      } else if (MODE == kDHidden) {
        float dw = 0.f;
        for (int chunk = 0; chunk < gu_total; ++chunk, ++gu_chunks) {
          const uint32_t set = gu_chunks & 1u;
          const bool here =
              ptx::mbar_wait(ptx::smem_u32(&ctrl->gu_full[set]), (gu_chunks >> 1) & 1u, abort_flag, p.timeout_ns);
          if (epi_tid == 0) ptx::tma_store_wait_read<1>();
          if (!ptx::named_barrier_all(kEpiBarrier, kEpiThreads, here)) {
            ok = false;
            break;
          }
          const uint32_t buf = smem_out + (stores & 1u) * kBoxBytes;
          const uint32_t gu = smem_gu + set * (2 * kBoxBytes) + stage_row;
          ptx::tmem_ld_32x32(t_acc + chunk * 32, r);
          ptx::tmem_ld_wait();
#pragma unroll
          for (uint32_t half = 0; half < 2; ++half) {
#pragma unroll
            for (uint32_t piece = 0; piece < 4; ++piece) {
              // four hidden columns: eight products, eight gradients, 16 bytes of output
              uint32_t o[4];
#pragma unroll
              for (uint32_t q = 0; q < 2; ++q) {
                const float4 v = ld_shared_v4(gu + half * kBoxBytes + ((piece * 2 + q) ^ sw) * 16);
                const int j = half * 16 + piece * 4 + q * 2;
                const float d0 = __uint_as_float(r[j]), d1 = __uint_as_float(r[j + 1]);
                const float2 a0 = gate_act(v.x, p.activation), a1 = gate_act(v.z, p.activation);
                // (columns past the last are zero in both operands)
                dw += d0 * (a0.x * v.y) + d1 * (a1.x * v.w);
                o[q * 2] = live ? pack2<BF16>(weight * d0 * v.y * a0.y, weight * d0 * a0.x) : 0u;
                o[q * 2 + 1] = live ? pack2<BF16>(weight * d1 * v.w * a1.y, weight * d1 * a1.x) : 0u;
              }
              st_shared_v4(buf + stage_row + ((half * 4 + piece) ^ sw) * 16, o[0], o[1], o[2], o[3]);
            }
          }
          end();
          if (epi_tid == 0) {
            ptx::tma_store_2d(&tmap_c, 2 * (un.col0 + chunk * 32), row0, buf);
            ptx::tma_store_commit();
            // (the barrier in end() says that everyone has read this chunk)
            if (chunk + 2 < gu_total) fetch_gu(chunk + 2, gu_chunks + 2);
          }
        }
        if (!ok) break;
        if (live) p.dw_part[static_cast<long long>(row0 + row_in_tile) * p.tiles_n + un.tile_col] = dw;
      } else {
        for (int col = 0; col < TILE_N; col += 64) {
          if (un.col0 + col >= p.cols) break;
          const uint32_t buf = begin();
#pragma unroll
          for (int sub = 0; sub < 2; ++sub) {
            ptx::tmem_ld_32x32(t_acc + col + sub * 32, r);
            ptx::tmem_ld_wait();
#pragma unroll
            for (uint32_t piece = 0; piece < 4; ++piece)
              st_shared_v4(buf + stage_row + ((sub * 4 + piece) ^ sw) * 16,
                           pack2<BF16>(__uint_as_float(r[piece * 8]), __uint_as_float(r[piece * 8 + 1])),
                           pack2<BF16>(__uint_as_float(r[piece * 8 + 2]), __uint_as_float(r[piece * 8 + 3])),
                           pack2<BF16>(__uint_as_float(r[piece * 8 + 4]), __uint_as_float(r[piece * 8 + 5])),
                           pack2<BF16>(__uint_as_float(r[piece * 8 + 6]), __uint_as_float(r[piece * 8 + 7])));
          }
          end();
          // (the second CTA of a pair may lie past the last row altogether)
          if (epi_tid == 0 && row0 < p.m) {
            ptx::tma_store_3d(&tmap_c, un.col0 + col, row0, un.expert, buf);
            ptx::tma_store_commit();
          }
        }
      }
      // All loads of this accumulator are complete: hand the TMEM buffer back.
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        const uint32_t te = ptx::smem_u32(&ctrl->tmem_empty[acc]);
        if (leader)
          ptx::mbar_arrive(te);
        else
          ptx::mbar_arrive_cluster(ptx::mapa(te, 0));
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1u;
      }
    }
    if (epi_tid == 0) ptx::tma_store_wait_all<0>();
    if (!ok && lane == 0 && p.status != nullptr) atomicCAS(p.status, 0, kAbortEpilogue);
  }

  // ------------------------------------------------------------------ teardown
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (ctrl->abort != 0) {
    // A wait gave up: let copies and MMAs still in flight drain before shared memory and TMEM
    // are released (bounded: about a millisecond).
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
  __syncwarp();
  if (CTA_GROUP == 2) {
    ptx::cluster_arrive();
    ptx::cluster_wait();
  }
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<CTA_GROUP>(tmem_base, 2 * TILE_N);
  }
}

// ----------------------------------------------------------------------- rows in and out of order

// out[pos[t, s]] = in[t] for every slot: a 16-byte piece of a token is read once and stored top_k
// times.  The blocks from `copy_blocks` on (where there are any) clear an expert's rows from its
// last to the next multiple of 64 each, which products over K = rows read.
__global__ void __launch_bounds__(256) permute_kernel(const Plan plan, const uint4* in, long long ld_in, uint4* out,
                                                      int tokens, int top_k, int vectors, int copy_blocks) {
  dependency_wait();
  dependency_release();
  if (static_cast<int>(blockIdx.x) >= copy_blocks) {
    const int e = blockIdx.x - copy_blocks;
    const int count = plan.count[e];
    const long long first = static_cast<long long>(plan.start[e] + count) * vectors;
    const int clear = ((count + kTileK - 1) / kTileK * kTileK - count) * vectors;
    for (int i = threadIdx.x; i < clear; i += 256) out[first + i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const long long total = static_cast<long long>(tokens) * vectors;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += copy_blocks * 256ll) {
    const int t = static_cast<int>(i / vectors);
    const int c = static_cast<int>(i - static_cast<long long>(t) * vectors);
    const uint4 v = in[t * ld_in + c];
    for (int s = 0; s < top_k; ++s) {
      const int row = plan.pos[static_cast<long long>(t) * top_k + s];
      if (row >= 0) out[static_cast<long long>(row) * vectors + c] = v;
    }
  }
}

// out[t] = sum over slots of part[pos[t, s]], in slot order; slots without an expert add nothing.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const float* part, const int* pos, T* out, long long ld_out,
                                                      int tokens, int top_k, int cols) {
  dependency_wait();
  dependency_release();
  const int vectors = cols >> 3;
  const long long total = static_cast<long long>(tokens) * vectors;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const int t = static_cast<int>(i / vectors);
    const int c = static_cast<int>(i - static_cast<long long>(t) * vectors) * 8;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < top_k; ++s) {
      const int row = pos[static_cast<long long>(t) * top_k + s];
      if (row < 0) continue;
      float v[8];
      elem::load<float, 8>(part + static_cast<long long>(row) * cols + c, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += v[j];
    }
    elem::store<T, 8>(out + t * ld_out + c, sum);
  }
}

// dweights[pair] = sum over column tiles of the pair's row, in order.
__global__ void __launch_bounds__(256) weight_grad_kernel(const float* dw_part, const int* pos, float* dweights,
                                                          int pairs, int tiles_n) {
  dependency_wait();
  dependency_release();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= pairs) return;
  const int row = pos[i];
  float sum = 0.f;
  if (row >= 0)
    for (int c = 0; c < tiles_n; ++c) sum += dw_part[static_cast<long long>(row) * tiles_n + c];
  dweights[i] = sum;
}

// ------------------------------------------------------------------------------------- host

inline int cdiv(int a, int b) { return (a + b - 1) / b; }
inline int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Sizes and offsets of one problem.
struct Layout {
  int cta_group, tile_rows, pairs, max_tiles;
  int64_t max_rows;
  int chunk, chunks;
  // forward: everything in `saved` when training (and the rest in the workspace)
  int64_t off_tiles, off_count, off_start, off_tile_expert, off_row_token, off_row_weight, off_pos, plan_bytes;
  bool gather;         // the copy engine picks the rows of x
  int64_t hidden_bytes, gu_bytes, part_bytes, chunk_bytes, x_bytes;
  int64_t dgu_bytes, dx_bytes, dw_bytes, dy_bytes;
};

int moe_check(const tnx_moe_problem* p) {
  if (p == nullptr) {
    set_error("problem is NULL");
    return TNX_ERR_INVALID;
  }
  if (p->dtype != TNX_F16 && p->dtype != TNX_BF16) {
    set_error("the experts' products take fp16 or bf16 operands");
    return TNX_ERR_INVALID;
  }
  if (p->activation < TNX_EPI_GLU_LINEAR || p->activation > TNX_EPI_GLU_SIGMOID) {
    set_error("activation must be TNX_EPI_GLU_LINEAR, _SILU or _SIGMOID, got %d", p->activation);
    return TNX_ERR_INVALID;
  }
  if (p->tokens < 0 || p->experts < 1 || p->experts > kMaxExperts || p->top_k < 1 ||
      static_cast<int64_t>(p->tokens) * p->top_k > (1 << 28)) {
    set_error("needs tokens >= 0, 1 <= experts <= %d, top_k >= 1 and at most 2^28 (token, slot) pairs "
              "(got %d tokens, %d experts, top_k %d)", kMaxExperts, p->tokens, p->experts, p->top_k);
    return TNX_ERR_INVALID;
  }
  if (p->d_model < 8 || p->d_ff < 8 || p->n_out < 8 || (p->d_model % 8) || (p->d_ff % 8) || (p->n_out % 8) ||
      p->d_model > (1 << 20) || p->d_ff > (1 << 20) || p->n_out > (1 << 20)) {
    set_error("d_model, d_ff and n_out must be positive multiples of 8 up to 2^20 (got %d, %d, %d)", p->d_model,
              p->d_ff, p->n_out);
    return TNX_ERR_INVALID;
  }
  if (p->stride_x < p->d_model || p->stride_w12k < 2ll * p->d_ff || p->stride_w3k < p->n_out ||
      p->stride_y < p->n_out || (p->stride_x % 8) || (p->stride_w12k % 8) || (p->stride_w3k % 8) ||
      (p->stride_w12e % 8) || (p->stride_w3e % 8) || (p->stride_y % 8) ||
      p->stride_w12e / p->stride_w12k < p->d_model || p->stride_w3e / p->stride_w3k < p->d_ff) {
    set_error("pitches of rows and of experts must cover them and be multiples of 8 elements (16 bytes)");
    return TNX_ERR_INVALID;
  }
  // (tile numbers are 32-bit; the smallest tiles are 128 rows x 128 columns)
  const int64_t row_tiles = static_cast<int64_t>(p->tokens) * p->top_k / kRows + p->experts;
  const int64_t widest = p->d_model > 2 * p->d_ff ? p->d_model : 2 * p->d_ff;
  const int64_t weight_tiles = static_cast<int64_t>(p->experts) * (widest / 128 + 1);
  if ((row_tiles > weight_tiles ? row_tiles : weight_tiles) * ((widest > p->n_out ? widest : p->n_out) / 128 + 1) >
      (1 << 30)) {
    set_error("problem has too many tiles");
    return TNX_ERR_INVALID;
  }
  return TNX_OK;
}

Layout lay_out_problem(const tnx_moe_problem& p) {
  Layout l = {};
  l.pairs = p.tokens * p.top_k;
  // Pairs of CTAs (256-row tiles) halve the weight traffic per row but pad an expert to 256 rows.
  l.cta_group = l.pairs / p.experts >= 384 ? 2 : 1;
  l.tile_rows = kRows * l.cta_group;
  l.max_tiles = l.pairs / l.tile_rows + (l.pairs < p.experts ? l.pairs : p.experts);
  l.max_rows = static_cast<int64_t>(l.max_tiles) * l.tile_rows;
  if (l.pairs <= kSmallPairs) {
    l.chunk = cdiv(cdiv(l.pairs, kSmallWarps), 32) * 32;
    l.chunks = kSmallWarps;
  } else {
    l.chunk = kChunkPairs;
    l.chunks = cdiv(l.pairs, kChunkPairs);
    l.chunk_bytes = align256(4ll * l.chunks * p.experts);
  }
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  l.off_tiles = take(4);
  l.off_count = take(4ll * p.experts);
  l.off_start = take(4ll * p.experts);
  l.off_tile_expert = take(4ll * l.max_tiles);
  l.off_row_token = take(4 * l.max_rows);
  l.off_row_weight = take(4 * l.max_rows);
  l.off_pos = take(4ll * l.pairs);
  l.plan_bytes = at;
  // (a training step needs the rows in order for the weights' gradients anyway)
  l.gather = !p.train && l.pairs / p.experts <= 32;
  l.x_bytes = l.gather ? 0 : align256(l.max_rows * p.d_model * 2);
  l.dy_bytes = align256(l.max_rows * p.n_out * 2);
  l.hidden_bytes = align256(l.max_rows * p.d_ff * 2);
  l.gu_bytes = align256(l.max_rows * p.d_ff * 8);
  l.part_bytes = align256(l.max_rows * p.n_out * 4);
  l.dgu_bytes = align256(l.max_rows * p.d_ff * 4);
  l.dx_bytes = align256(l.max_rows * p.d_model * 4);
  l.dw_bytes = align256(l.max_rows * cdiv(p.d_ff, tile_n(kDHidden, l.cta_group)) * 4);
  return l;
}

Plan plan_at(const Layout& l, void* base) {
  char* b = static_cast<char*>(base);
  Plan q;
  q.tiles = reinterpret_cast<int*>(b + l.off_tiles);
  q.count = reinterpret_cast<int*>(b + l.off_count);
  q.start = reinterpret_cast<int*>(b + l.off_start);
  q.tile_expert = reinterpret_cast<int*>(b + l.off_tile_expert);
  q.row_token = reinterpret_cast<int*>(b + l.off_row_token);
  q.row_weight = reinterpret_cast<float*>(b + l.off_row_weight);
  q.pos = reinterpret_cast<int*>(b + l.off_pos);
  return q;
}

int cuda_failed(const char* what, cudaError_t e) {
  set_error("%s: %s", what, cudaGetErrorString(e));
  (void)cudaGetLastError();
  return TNX_ERR_CUDA;
}

// Opts a kernel into `bytes` of dynamic shared memory, once per (kernel, device).
cudaError_t allow_smem(const void* fn, int bytes) {
  constexpr int kSlots = 64;
  static std::mutex mu;
  static std::pair<const void*, int> done[kSlots];
  static int used = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < used; ++i)
    if (done[i].first == fn && done[i].second == dev) return cudaSuccess;
  e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && used < kSlots) done[used++] = {fn, dev};
  return e;
}

// Launches with programmatic stream serialization (every kernel here calls dependency_wait()).
template <typename... KArgs, typename... Args>
int launch(const char* what, void (*fn)(KArgs...), int grid, int block, int smem, int cluster, cudaStream_t stream,
           Args... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  lc.blockDim = dim3(static_cast<unsigned>(block), 1, 1);
  lc.dynamicSmemBytes = static_cast<size_t>(smem);
  lc.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[n].val.programmaticStreamSerializationAllowed = 1;
  ++n;
  lc.attrs = attr;
  lc.numAttrs = static_cast<unsigned>(n);
  const cudaError_t e = cudaLaunchKernelEx(&lc, fn, args...);
  return e == cudaSuccess ? TNX_OK : cuda_failed(what, e);
}

template <int MODE, int CTA_GROUP>
int launch_gemm(int dtype, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c, const CUtensorMap& gu,
                GemmParams p, int64_t units, cudaStream_t stream) {
  constexpr int n = tile_n(MODE, CTA_GROUP);
  constexpr int stage_bytes = (kRows + n / CTA_GROUP) * kTileK * 2;
  constexpr int fixed = staging_boxes(MODE) * kBoxBytes + kCtrlBytes + kAlignSlack;
  constexpr int fit = (kMaxDynamicSmem - fixed) / stage_bytes;
  constexpr int stages = fit > kMaxStages ? kMaxStages : fit;
  static_assert(stages >= 3, "too little shared memory for the ring");
  p.stages = stages;
  p.tile_rows = kRows * CTA_GROUP;
  auto fn = dtype == TNX_BF16 ? moe_gemm_kernel<MODE, CTA_GROUP, true> : moe_gemm_kernel<MODE, CTA_GROUP, false>;
  const int smem = stages * stage_bytes + fixed;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(fn), kMaxDynamicSmem);
  if (e != cudaSuccess) return cuda_failed("experts' products: shared memory", e);
  const int most = sm_count() / CTA_GROUP;
  const int clusters = units < most ? static_cast<int>(units) : most;
  if (clusters < 1) return TNX_OK;
  return launch("experts' products", fn, clusters * CTA_GROUP, kThreads, smem, CTA_GROUP, stream, a, b, c, gu, p);
}
template <int MODE>
int launch_gemm(const Layout& l, int dtype, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& c,
                const CUtensorMap& gu, const GemmParams& p, int64_t units, cudaStream_t stream) {
  return l.cta_group == 2 ? launch_gemm<MODE, 2>(dtype, a, b, c, gu, p, units, stream)
                          : launch_gemm<MODE, 1>(dtype, a, b, c, gu, p, units, stream);
}

int run_plan(const tnx_moe_problem& p, const Layout& l, const Plan& plan, const void* ids, const float* weights,
             void* scratch, cudaStream_t stream) {
  PlanParams q = {};
  q.plan = plan;
  q.ids = ids;
  q.weights = weights;
  q.wide = p.wide_ids;
  q.experts = p.experts;
  q.top_k = p.top_k;
  q.pairs = l.pairs;
  q.tile_rows = l.tile_rows;
  q.chunk = l.chunk;
  q.chunks = l.chunks;
  q.chunk_counts = static_cast<int*>(scratch);
  if (l.pairs <= kSmallPairs) {
    const int smem = static_cast<int>(sizeof(SmallPlanSmem));
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(plan_small_kernel), smem);
    if (e != cudaSuccess) return cuda_failed("routing plan: shared memory", e);
    return launch("routing plan", plan_small_kernel, 1, kSmallWarps * 32, smem, 1, stream, q);
  }
  const int blocks = cdiv(l.chunks, kChunkWarps);
  int rc = launch("routing plan (count)", plan_count_kernel, blocks, kChunkWarps * 32, 0, 1, stream, q);
  if (rc == TNX_OK) rc = launch("routing plan (scan)", plan_scan_kernel, 1, 1024, 0, 1, stream, q);
  if (rc == TNX_OK) rc = launch("routing plan (place)", plan_place_kernel, blocks, kChunkWarps * 32, 0, 1, stream, q);
  return rc;
}

// Rows of `in` [tokens, cols] in expert order.
int run_permute(const tnx_moe_problem& p, const Plan& plan, const void* in, int64_t ld_in, void* out, int cols,
                bool clear, cudaStream_t stream) {
  const int vectors = cols / 8;
  const int64_t blocks = (static_cast<int64_t>(p.tokens) * vectors + 255) / 256;
  const int most = 16 * sm_count();
  const int grid = blocks < most ? static_cast<int>(blocks) : most;
  return launch("rows in expert order", permute_kernel, grid + (clear ? p.experts : 0), 256, 0, 1, stream, plan,
                static_cast<const uint4*>(in), static_cast<long long>(ld_in / 8), static_cast<uint4*>(out), p.tokens,
                p.top_k, vectors, grid);
}

int run_combine(int dtype, const float* part, const int* pos, void* out, int64_t ld_out, int tokens, int top_k,
                int cols, cudaStream_t stream) {
  const int64_t blocks = (static_cast<int64_t>(tokens) * (cols / 8) + 255) / 256;
  const int most = 16 * sm_count();
  const int grid = blocks < most ? static_cast<int>(blocks) : most;
  if (dtype == TNX_BF16)
    return launch("combining experts", combine_kernel<__nv_bfloat16>, grid, 256, 0, 1, stream, part, pos,
                  static_cast<__nv_bfloat16*>(out), static_cast<long long>(ld_out), tokens, top_k, cols);
  return launch("combining experts", combine_kernel<__half>, grid, 256, 0, 1, stream, part, pos,
                static_cast<__half*>(out), static_cast<long long>(ld_out), tokens, top_k, cols);
}

GemmParams gemm_params(const tnx_moe_problem& p, const Plan& plan, int32_t* status) {
  GemmParams g = {};
  g.plan = plan;
  g.experts = p.experts;
  g.activation = p.activation;
  g.band = 8;
  g.status = status;
  g.timeout_ns = bounded_wait_limit_ns();
  return g;
}

bool misaligned(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15u) != 0; }
bool off256(const void* a) { return (reinterpret_cast<uintptr_t>(a) & 255u) != 0; }

}  // namespace
}  // namespace tnx

extern "C" {

int tnx_moe_query(const tnx_moe_problem* problem, tnx_moe_resources* out) {
  using namespace tnx;
  if (out == nullptr) {
    set_error("out is NULL");
    return TNX_ERR_INVALID;
  }
  const int rc = moe_check(problem);
  if (rc != TNX_OK) return rc;
  const Layout l = lay_out_problem(*problem);
  out->tile_rows = l.tile_rows;
  out->max_tiles = l.max_tiles;
  const int64_t keep = l.plan_bytes + l.hidden_bytes;
  out->saved_bytes = keep + l.gu_bytes;
  out->workspace_bytes = l.part_bytes + l.chunk_bytes + l.x_bytes + (problem->train ? 0 : keep);
  out->backward_workspace_bytes = l.dgu_bytes + l.dx_bytes + l.dw_bytes + l.x_bytes + l.dy_bytes;
  return TNX_OK;
}

int tnx_moe_swiglu(const tnx_moe_problem* problem, const void* x, const void* w12, const void* w3, const void* ids,
                   const float* weights, void* y, void* saved, void* workspace, size_t workspace_bytes,
                   int32_t* status_word, void* stream) {
  using namespace tnx;
  tnx_moe_resources res;
  int rc = tnx_moe_query(problem, &res);
  if (rc != TNX_OK) return rc;
  const tnx_moe_problem& p = *problem;
  if (p.tokens == 0) return TNX_OK;
  if (x == nullptr || w12 == nullptr || w3 == nullptr || ids == nullptr || weights == nullptr || y == nullptr ||
      (p.train && saved == nullptr)) {
    set_error("NULL operand pointer");
    return TNX_ERR_INVALID;
  }
  if (misaligned(x) || misaligned(w12) || misaligned(w3) || misaligned(y)) {
    set_error("x, w12, w3 and y must be 16-byte aligned");
    return TNX_ERR_INVALID;
  }
  if (workspace == nullptr || workspace_bytes < static_cast<size_t>(res.workspace_bytes) || off256(workspace) ||
      (p.train && off256(saved))) {
    set_error("the experts' products need a workspace of %lld bytes, 256-byte aligned like the saved tensors",
              static_cast<long long>(res.workspace_bytes));
    return TNX_ERR_INVALID;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Layout l = lay_out_problem(p);
  char* ws = static_cast<char*>(workspace);
  float* part = reinterpret_cast<float*>(ws);
  void* chunk_counts = ws + l.part_bytes;
  void* xp = ws + l.part_bytes + l.chunk_bytes;
  char* keep = p.train ? static_cast<char*>(saved) : ws + l.part_bytes + l.chunk_bytes + l.x_bytes;
  const Plan plan = plan_at(l, keep);
  void* hidden = keep + l.plan_bytes;
  void* gu = p.train ? keep + l.plan_bytes + l.hidden_bytes : nullptr;

  rc = run_plan(p, l, plan, ids, weights, chunk_counts, s);
  if (rc == TNX_OK && !l.gather) rc = run_permute(p, plan, x, p.stride_x, xp, p.d_model, false, s);
  if (rc != TNX_OK) return rc;

  // H = w * act(x W1) * (x W2)
  GemmParams g = gemm_params(p, plan, status_word);
  g.num_kb = cdiv(p.d_model, kTileK);
  g.cols = 2 * p.d_ff;
  g.tiles_n = cdiv(g.cols, 256);
  g.save_gu = p.train;
  CUtensorMap ta, tb, tc, tgu;
  rc = l.gather ? make_tmap_2d(&ta, x, p.dtype, p.d_model, p.tokens, p.stride_x, 64, 1, true)
                : make_tmap_2d(&ta, xp, p.dtype, p.d_model, l.max_rows, p.d_model, 64, 32, true);
  if (rc == TNX_OK)
    rc = make_tmap_3d(&tb, w12, p.dtype, 2ll * p.d_ff, p.d_model, p.experts, p.stride_w12k, p.stride_w12e, 64, kTileK, true);
  if (rc == TNX_OK) rc = make_tmap_2d(&tc, hidden, p.dtype, p.d_ff, l.max_rows, p.d_ff, 64, kRows, false);
  tgu = tc;
  if (rc == TNX_OK && p.train)
    rc = make_tmap_2d(&tgu, gu, TNX_F32, 2ll * p.d_ff, l.max_rows, 2ll * p.d_ff, 32, kRows, false);
  if (rc != TNX_OK) return rc;
  const int64_t units = static_cast<int64_t>(l.max_tiles) * g.tiles_n;
  rc = l.gather ? launch_gemm<kGateUpGather>(l, p.dtype, ta, tb, tc, tgu, g, units, s)
                : launch_gemm<kGateUp>(l, p.dtype, ta, tb, tc, tgu, g, units, s);
  if (rc != TNX_OK) return rc;

  // O = H W3
  g.num_kb = cdiv(p.d_ff, kTileK);
  g.cols = p.n_out;
  g.tiles_n = cdiv(g.cols, 256);
  g.part = part;
  rc = make_tmap_2d(&ta, hidden, p.dtype, p.d_ff, l.max_rows, p.d_ff, 64, 32, true);
  if (rc == TNX_OK)
    rc = make_tmap_3d(&tb, w3, p.dtype, p.n_out, p.d_ff, p.experts, p.stride_w3k, p.stride_w3e, 64, kTileK, true);
  if (rc == TNX_OK) rc = make_tmap_2d(&tc, part, TNX_F32, p.n_out, l.max_rows, p.n_out, 32, kRows, false);
  if (rc != TNX_OK) return rc;
  rc = launch_gemm<kDown>(l, p.dtype, ta, tb, tc, tc, g, static_cast<int64_t>(l.max_tiles) * g.tiles_n, s);
  if (rc != TNX_OK) return rc;
  return run_combine(p.dtype, part, plan.pos, y, p.stride_y, p.tokens, p.top_k, p.n_out, s);
}

int tnx_moe_swiglu_backward(const tnx_moe_problem* problem, const void* dy, int64_t stride_dy, const void* x,
                            const void* w12, const void* w3, const void* saved, void* dx, void* dw12, void* dw3,
                            float* dweights, void* workspace, size_t workspace_bytes, int32_t* status_word,
                            void* stream) {
  using namespace tnx;
  tnx_moe_resources res;
  int rc = tnx_moe_query(problem, &res);
  if (rc != TNX_OK) return rc;
  const tnx_moe_problem& p = *problem;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t w12_bytes = 4ll * p.experts * p.d_model * p.d_ff, w3_bytes = 2ll * p.experts * p.d_ff * p.n_out;
  if (p.tokens == 0) {  // no rows: the weights' gradients are zero
    cudaError_t e = cudaSuccess;
    if (dw12 != nullptr) e = cudaMemsetAsync(dw12, 0, static_cast<size_t>(w12_bytes), s);
    if (e == cudaSuccess && dw3 != nullptr) e = cudaMemsetAsync(dw3, 0, static_cast<size_t>(w3_bytes), s);
    return e == cudaSuccess ? TNX_OK : cuda_failed("experts' gradients", e);
  }
  if (dy == nullptr || x == nullptr || w12 == nullptr || w3 == nullptr || saved == nullptr) {
    set_error("NULL operand pointer");
    return TNX_ERR_INVALID;
  }
  if (misaligned(dy) || misaligned(x) || misaligned(w12) || misaligned(w3) || misaligned(dx) || misaligned(dw12) ||
      misaligned(dw3) || stride_dy < p.n_out || stride_dy % 8) {
    set_error("operands and gradients must be 16-byte aligned and dy's row pitch a multiple of 8 that covers n_out");
    return TNX_ERR_INVALID;
  }
  if (workspace == nullptr || workspace_bytes < static_cast<size_t>(res.backward_workspace_bytes) ||
      off256(workspace) || off256(saved)) {
    set_error("the experts' gradients need a workspace of %lld bytes, 256-byte aligned like the saved tensors",
              static_cast<long long>(res.backward_workspace_bytes));
    return TNX_ERR_INVALID;
  }
  const Layout l = lay_out_problem(p);
  char* keep = static_cast<char*>(const_cast<void*>(saved));
  const Plan plan = plan_at(l, keep);
  void* hidden = keep + l.plan_bytes;
  void* gu = keep + l.plan_bytes + l.hidden_bytes;
  char* ws = static_cast<char*>(workspace);
  void* dgu = ws;
  float* dx_part = reinterpret_cast<float*>(ws + l.dgu_bytes);
  float* dw_part = reinterpret_cast<float*>(ws + l.dgu_bytes + l.dx_bytes);
  void* xp = ws + l.dgu_bytes + l.dx_bytes + l.dw_bytes;
  void* dyp = ws + l.dgu_bytes + l.dx_bytes + l.dw_bytes + l.x_bytes;
  const int64_t two_f = 2ll * p.d_ff;
  const bool hidden_grad = dx != nullptr || dw12 != nullptr || dweights != nullptr;
  if (hidden_grad || dw3 != nullptr) rc = run_permute(p, plan, dy, stride_dy, dyp, p.n_out, true, s);
  if (rc == TNX_OK && dw12 != nullptr) rc = run_permute(p, plan, x, p.stride_x, xp, p.d_model, true, s);
  if (rc != TNX_OK) return rc;

  // dH = dy W3^T; dGU and the routing weights' gradient from it
  GemmParams g = gemm_params(p, plan, status_word);
  CUtensorMap ta, tb, tc, tgu;
  if (hidden_grad) {
    const int n = tile_n(kDHidden, l.cta_group);
    g.num_kb = cdiv(p.n_out, kTileK);
    g.cols = p.d_ff;
    g.tiles_n = cdiv(g.cols, n);
    g.dw_part = dw_part;
    rc = make_tmap_2d(&ta, dyp, p.dtype, p.n_out, l.max_rows, p.n_out, 64, 32, true);
    if (rc == TNX_OK)
      rc = make_tmap_3d(&tb, w3, p.dtype, p.n_out, p.d_ff, p.experts, p.stride_w3k, p.stride_w3e, 64,
                        n / l.cta_group, true);
    if (rc == TNX_OK) rc = make_tmap_2d(&tc, dgu, p.dtype, two_f, l.max_rows, two_f, 64, kRows, false);
    if (rc == TNX_OK) rc = make_tmap_2d(&tgu, gu, TNX_F32, two_f, l.max_rows, two_f, 32, kRows, true);
    if (rc != TNX_OK) return rc;
    rc = launch_gemm<kDHidden>(l, p.dtype, ta, tb, tc, tgu, g, static_cast<int64_t>(l.max_tiles) * g.tiles_n, s);
    if (rc != TNX_OK) return rc;
    if (dweights != nullptr) {
      rc = launch("routing weights' gradient", weight_grad_kernel, cdiv(l.pairs, 256), 256, 0, 1, s,
                  static_cast<const float*>(dw_part), static_cast<const int*>(plan.pos), dweights, l.pairs, g.tiles_n);
      if (rc != TNX_OK) return rc;
    }
  }
  if (dx != nullptr) {
    g.num_kb = cdiv(static_cast<int>(two_f), kTileK);
    g.cols = p.d_model;
    g.tiles_n = cdiv(g.cols, 256);
    g.part = dx_part;
    rc = make_tmap_2d(&ta, dgu, p.dtype, two_f, l.max_rows, two_f, 64, 32, true);
    if (rc == TNX_OK)
      rc = make_tmap_3d(&tb, w12, p.dtype, two_f, p.d_model, p.experts, p.stride_w12k, p.stride_w12e, 64,
                        256 / l.cta_group, true);
    if (rc == TNX_OK) rc = make_tmap_2d(&tc, dx_part, TNX_F32, p.d_model, l.max_rows, p.d_model, 32, kRows, false);
    if (rc != TNX_OK) return rc;
    rc = launch_gemm<kDX>(l, p.dtype, ta, tb, tc, tc, g, static_cast<int64_t>(l.max_tiles) * g.tiles_n, s);
    if (rc == TNX_OK)
      rc = run_combine(p.dtype, dx_part, plan.pos, dx, p.d_model, p.tokens, p.top_k, p.d_model, s);
    if (rc != TNX_OK) return rc;
  }
  if (dw12 != nullptr) {
    g.m = p.d_model;
    g.tiles_m = cdiv(p.d_model, l.tile_rows);
    g.cols = static_cast<int>(two_f);
    g.tiles_n = cdiv(g.cols, 256);
    rc = make_tmap_2d(&ta, xp, p.dtype, p.d_model, l.max_rows, p.d_model, 64, kTileK, true);
    if (rc == TNX_OK) rc = make_tmap_2d(&tb, dgu, p.dtype, two_f, l.max_rows, two_f, 64, kTileK, true);
    if (rc == TNX_OK)
      rc = make_tmap_3d(&tc, dw12, p.dtype, two_f, p.d_model, p.experts, two_f, two_f * p.d_model, 64, kRows, false);
    if (rc != TNX_OK) return rc;
    rc = launch_gemm<kDW12>(l, p.dtype, ta, tb, tc, tc, g, static_cast<int64_t>(p.experts) * g.tiles_m * g.tiles_n, s);
    if (rc != TNX_OK) return rc;
  }
  if (dw3 != nullptr) {
    g.m = p.d_ff;
    g.tiles_m = cdiv(p.d_ff, l.tile_rows);
    g.cols = p.n_out;
    g.tiles_n = cdiv(g.cols, 256);
    rc = make_tmap_2d(&ta, hidden, p.dtype, p.d_ff, l.max_rows, p.d_ff, 64, kTileK, true);
    if (rc == TNX_OK) rc = make_tmap_2d(&tb, dyp, p.dtype, p.n_out, l.max_rows, p.n_out, 64, kTileK, true);
    if (rc == TNX_OK)
      rc = make_tmap_3d(&tc, dw3, p.dtype, p.n_out, p.d_ff, p.experts, p.n_out, static_cast<int64_t>(p.n_out) * p.d_ff,
                        64, kRows, false);
    if (rc != TNX_OK) return rc;
    rc = launch_gemm<kDW3>(l, p.dtype, ta, tb, tc, tc, g, static_cast<int64_t>(p.experts) * g.tiles_m * g.tiles_n, s);
    if (rc != TNX_OK) return rc;
  }
  return TNX_OK;
}

}  // extern "C"
