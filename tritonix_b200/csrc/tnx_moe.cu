// Experts' gated products for sm_100a:
//     y[t] = sum over slots s of  w[t, s] * ( act(x[t].W1[e]) * (x[t].W2[e]) ) . W3[e],  e = ids[t, s]
// with W12 = W1/W2 column-interleaved per expert, and its backward pass.
//
//  * A (token, slot) pair is a row of a grouped problem.  plan_* sorts the pairs by expert (stable:
//    rows of an expert keep the pairs' order, so every sum has a fixed order).  Nothing about the
//    routing is needed on the host.
//  * moe_rows_kernel multiplies rows by their expert's weights on CTA pairs (TMA -> shared memory ->
//    tcgen05 -> TMEM, the pipeline of the library's GEMM), with the WEIGHTS as the 256-row M
//    operand and the rows as N:  out^T = W^T rows^T.  N is a field of each instruction, so a tile
//    costs what its rows need, to a multiple of 32, instead of what 256 rows would (with rows as M
//    an expert's last tile is half empty on average: 12 % of the work at 64 experts and 65536
//    pairs, and under the power cap that is 12 % of the time), and all the rows of an expert with
//    up to 256 of them share one pass over its weights.  In the epilogue a lane then is a column
//    of the output and a register a row: every store is a coalesced row piece, straight from
//    registers, and unused rows cost nothing.
//        kGateUp  H = w * act(X W1) * (X W2)          X: the rows of x in expert order (kGateUpKeep: with
//                 the fp32 products kept for the backward pass)
//        kDown    O = H W3                            fp32, one row per pair
//        kDHidden dH = dY W3^T, then dGU and dw       dY: the rows of dy in expert order
//        kDX      O = dGU W12^T                       fp32, one row per pair
//    permute_kernel copies rows into expert order.  With few rows per expert the copy engine picks
//    them itself instead (kGateUpGather, tile::gather4, one lane per four rows): a gather of four
//    128-byte row pieces was measured to take about as long as a whole box of rows (40-75 cycles),
//    so many rows are better copied once (8192 tokens, 64 experts 2048/1024: gate/up product
//    1287 us gathered, 420 us copied), while a few rows cost nothing and save a launch.
//  * moe_wgrad_kernel computes X^T dGU and H^T dY per expert, K = the expert's rows.
//  * The routing weight is applied to the hidden activation before it is rounded: the rows of O
//    only need adding, and H is the very operand dW3 needs, so no value on the way is rounded
//    twice.  combine_kernel adds a token's rows of O in slot order (fp32) and rounds once.
//  * The gate/up products are kept in fp32 for the backward pass: rounding them to 16 bits would
//    add two more roundings to every gradient.
//  * The tensor cores add to an accumulator by cutting off, not rounding: a sum over K comes out
//    short by about 3e-9 K of its size.  That is nothing next to 16 bits, but the routing weights'
//    gradient is fp32 and takes it from both of its factors (measured: 6e-6 at K = 2048, 2.5e-5 at
//    8192).  So where a product feeds that gradient (kGateUpKeep, kDHidden) an accumulator only runs
//    over a few K blocks, and the epilogue adds those sums up in fp32.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <mutex>
#include <type_traits>
#include <utility>

#include "tnx_elem.cuh"
#include "tnx_internal.h"
#include "tnx_ptx.cuh"

namespace tnx {

namespace {

constexpr int kMaxExperts = 512;
constexpr int kRows = 128;       // rows of the M operand per CTA (TMEM lanes); a pair has 256
constexpr int kTileN = 256;      // columns of the N operand per pair at most
constexpr int kPad = 16;         // an expert's rows are padded to this: one MMA's K
constexpr int kTileK = 128;      // K elements per ring slot: two slabs of 64, a 128-byte swizzle row each.
                                 // (Slots of 64 wait and commit twice as often: the library's GEMM
                                 // loses 5-13 % with them at these sizes.)
constexpr int kSlab = 64;
constexpr int kThreads = 192;      // producer warp, MMA warp, four epilogue warps
constexpr int kRowsEpilogue = 16;  // epilogue warps of the rows' kernel: four per quarter of the TMEM lanes
constexpr int kRowsThreads = 64 + 32 * kRowsEpilogue;
constexpr int kAtomBytes = 128;
constexpr int kStageBytes = 2 * kRows * kTileK * 2;  // 128 rows of each operand
constexpr int kBoxBytes = 32 * kAtomBytes;           // an epilogue warp's box: 32 rows of 128 bytes
constexpr int kBoxes = 2;                            // staging boxes per epilogue warp
constexpr int kMaxStages = 8;
constexpr int kCtrlBytes = 512;
constexpr int kAlignSlack = 1024;

constexpr int kAbortProducer = 0x301;
constexpr int kAbortMma = 0x302;
constexpr int kAbortEpilogue = 0x303;

enum Mode { kGateUp, kGateUpGather, kGateUpKeep, kDown, kDHidden, kDX };
constexpr bool is_gate_up(int mode) { return mode == kGateUp || mode == kGateUpGather || mode == kGateUpKeep; }
// Products whose accumulators are added up in fp32 every so many K blocks.
constexpr bool sums_outside(int mode) { return mode == kGateUpKeep || mode == kDHidden; }
// (384 elements of bf16 or 256 of fp16 lose 1e-6 of that gradient, what fp32 loses by itself)
constexpr int sum_blocks(bool bf16) { return bf16 ? 3 : 2; }
// The sums of a tile are 64 values per epilogue thread, of which 16 stay in shared memory: held in
// registers altogether they spilled, and the spills' traffic took longer than the products (gate/up
// product of the training step of 4095 tokens, 16 experts 2048/2040: 389 us).  Tiles of 128 rows
// would need half of them, but fetch the weights twice as often: 395 us.
constexpr int kParkedRows = 16;

// Where the pairs went (device memory, written by the plan kernels).
struct Plan {
  int* tiles;        // [1] row tiles in use
  int* count;        // [experts] rows of an expert
  int* start;        // [experts] its first row (a multiple of kPad)
  int4* tile;        // [max_tiles] expert, first row, rows in use, rows up to the padding
  int* row_token;    // [max_rows] token of a row (rows in use only)
  float* row_weight; // [max_rows]
  int* pos;          // [pairs] row of a pair, -1 where its id is no expert
};

struct RowsMaps {
  CUtensorMap m[4];
};

struct RowsParams {
  Plan plan;
  int k;                             // K elements
  int num_kb, splits, kb_per_split;  // K blocks; slices of K, each with its own copy of O
  int cols;         // columns of the weight operand: 2 d_ff, n_out, d_ff or d_model
  int tiles_n;      // tiles of 256 of them
  int panels;       // the weights' map takes two 64-column panels at a time
  int band;         // row tiles per band of the tile order
  int activation;
  long long max_rows;
  void* out;        // H, dGU (16 bit) or O (fp32, [splits][max_rows][cols])
  float* gu;        // [max_rows][2 d_ff]: written by gate/up, read by kDHidden
  float* dw_part;   // kDHidden: [max_rows][dw_parts], one sum per 32 columns
  int dw_parts;
  int stages;
  int* status;
  unsigned long long timeout_ns;
};

struct WgradParams {
  Plan plan;
  int experts;
  int m, n;              // rows and columns of a weight's gradient
  int tiles_m, tiles_n;  // 256 x 256 tiles
  int panels_a, panels_b;  // whether the operands' maps take two 64-column panels at a time
  int stages;
  int* status;
  unsigned long long timeout_ns;
};

struct Ctrl {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
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
  int wide, experts, top_k, pairs;
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

// Given total[e] in shared memory: first row of every expert (in start[]) and the row tiles.  An
// expert's rows are cut into as few tiles of at most kTileN rows as possible, of equal size up to
// a multiple of 32.  All threads of the block take part; tile0[] is scratch.
__device__ __forceinline__ void lay_out(const PlanParams& p, const int* total, int* start, int* tile0) {
  const int tid = threadIdx.x;
  if (tid < 32) {
    int rows_before = 0, tiles_before = 0;
    for (int base = 0; base < p.experts; base += 32) {
      const int e = base + tid;
      const int count = e < p.experts ? total[e] : 0;
      const int rows = (count + kPad - 1) / kPad * kPad, tiles = (count + kTileN - 1) / kTileN;
      int row_sum = rows, tile_sum = tiles;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int r = __shfl_up_sync(0xffffffffu, row_sum, o), t = __shfl_up_sync(0xffffffffu, tile_sum, o);
        if (tid >= o) {
          row_sum += r;
          tile_sum += t;
        }
      }
      if (e < p.experts) {
        start[e] = rows_before + row_sum - rows;
        tile0[e] = tiles_before + tile_sum - tiles;
      }
      rows_before += __shfl_sync(0xffffffffu, row_sum, 31);
      tiles_before += __shfl_sync(0xffffffffu, tile_sum, 31);
    }
    if (tid == 0) *p.plan.tiles = tiles_before;
  }
  __syncthreads();
  for (int e = tid; e < p.experts; e += blockDim.x) {
    const int count = total[e];
    p.plan.count[e] = count;
    p.plan.start[e] = start[e];
    const int tiles = (count + kTileN - 1) / kTileN;
    const int size = tiles > 0 ? ((count + tiles - 1) / tiles + 31) / 32 * 32 : 0;
    for (int i = 0; i < tiles; ++i) {
      const int used = min(size, count - i * size);
      p.plan.tile[tile0[e] + i] = make_int4(e, start[e] + i * size, used, (used + kPad - 1) / kPad * kPad);
    }
  }
}

// Up to kSmallPairs pairs: the whole plan in one block of 32 warps.
constexpr int kSmallPairs = 8192;
constexpr int kSmallWarps = 32;
struct SmallPlanSmem {
  int next[kSmallWarps][kMaxExperts];
  int total[kMaxExperts];
  int start[kMaxExperts];
  int tile0[kMaxExperts];
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
  lay_out(p, s.total, s.start, s.tile0);
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
  __shared__ int total[kMaxExperts], start[kMaxExperts], tile0[kMaxExperts], strand_sum[1024];
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
  lay_out(p, total, start, tile0);
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
  if (activation == TNX_EPI_GLU_SILU) return make_float2(g * s, s + g * s * (1.f - s));
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
// Four rows of 64 elements each, picked by row number, for a CTA pair (see ptx::tma_load_2d_pair).
__device__ __forceinline__ void tma_gather4_pair(uint32_t dst, const void* tmap, int x, const int (&rows)[4],
                                                 uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(rows[0]), "r"(rows[1]), "r"(rows[2]), "r"(rows[3]),
      "r"(leader_bar)
      : "memory");
}

// What both kernels share: barriers, the pair's rendezvous, 512 columns of TMEM (two accumulators
// of 256), and their release.  Returns the TMEM base address.
__device__ __forceinline__ uint32_t set_up_pair(Ctrl* ctrl, int stages, int epilogue_warps, int warp) {
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(ptx::smem_u32(&ctrl->tmem_full[a]), 1);
      ptx::mbar_init(ptx::smem_u32(&ctrl->tmem_empty[a]), 2 * epilogue_warps);  // one arrive each
    }
    ctrl->abort = 0;
    ptx::fence_mbar_init();
  }
  __syncwarp();
  ptx::cluster_arrive();  // the peer's barriers must exist before anything signals them
  ptx::cluster_wait();
  if (warp == 1) {
    ptx::tmem_alloc<2>(ptx::smem_u32(&ctrl->tmem_base), 2 * kTileN);
    ptx::tmem_relinquish<2>();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  return ctrl->tmem_base;
}
__device__ __forceinline__ void tear_down_pair(Ctrl* ctrl, uint32_t tmem_base, int warp) {
  ptx::tc_fence_before_sync();
  __syncthreads();
  if (ctrl->abort != 0) {
    // A wait gave up: let copies and MMAs still in flight drain before shared memory and TMEM
    // are released (bounded: about a millisecond).
    const uint64_t t0 = ptx::globaltimer_ns();
    while (ptx::globaltimer_ns() - t0 < 1000000ull) __nanosleep(1000);
  }
  __syncwarp();
  ptx::cluster_arrive();
  ptx::cluster_wait();
  if (warp == 1) {
    __syncwarp();
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc<2>(tmem_base, 2 * kTileN);
  }
}
// An epilogue warp has read all it needs of accumulator `acc`.
__device__ __forceinline__ void release_accumulator(Ctrl* ctrl, int acc, bool leader, int lane) {
  ptx::tc_fence_before_sync();
  __syncwarp();
  if (lane == 0) {
    const uint32_t te = ptx::smem_u32(&ctrl->tmem_empty[acc]);
    if (leader)
      ptx::mbar_arrive(te);
    else
      ptx::mbar_arrive_cluster(ptx::mapa(te, 0));
  }
}
// Ring position / accumulator that advances with its phase bit.
struct Cursor {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++at == size) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// One tile: a row tile of an expert and 256 columns of its weights (and a slice of K).
struct Unit {
  int expert, row0, used, padded;  // as in Plan::tile
  int n;                           // `used` up to a multiple of 32: N of the product
  int col0;
  int slice, kb0, num_kb;
};
template <int MODE>
__device__ __forceinline__ Unit decode_unit(const RowsParams& p, int u, int num_tiles) {
  Unit r;
  r.slice = 0;
  if (MODE == kDown || MODE == kDX) {
    r.slice = u % p.splits;
    u /= p.splits;
  }
  // bands of `band` row tiles, column tile by column tile inside a band: the pairs at work share the
  // weight tiles of few experts and the rows of one band through L2
  const int full = p.band * p.tiles_n;
  const int b = u / full;
  const int rem = u - b * full;
  const int rows = min(p.band, num_tiles - b * p.band);
  const int col = rem / rows;
  const int4 tile = p.plan.tile[b * p.band + (rem - col * rows)];
  r.expert = tile.x;
  r.row0 = tile.y;
  r.used = tile.z;
  r.padded = tile.w;
  r.n = (tile.z + 31) / 32 * 32;
  r.col0 = col * (2 * kRows);
  r.kb0 = r.slice * p.kb_per_split;
  r.num_kb = min(p.kb_per_split, p.num_kb - r.kb0);
  return r;
}

// Sum over the lanes of v[t] for every t, left in lane t.  31 exchanges: each halves the values a
// lane still carries.
__device__ __forceinline__ float transposed_sum(uint32_t (&v)[32], int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool upper = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const uint32_t give = upper ? v[i] : v[i + o];
      const float got = __uint_as_float(__shfl_xor_sync(0xffffffffu, give, o));
      v[i] = __float_as_uint(__uint_as_float(upper ? v[i + o] : v[i]) + got);
    }
  }
  return __uint_as_float(v[0]);
}

// What an epilogue warp reads from memory for 32 rows, before it needs it.
template <int MODE>
struct Prefetched {
  float weight = 0.f;  // routing weight of row j0 + lane, 0 for padding
  __device__ __forceinline__ void fetch(const RowsParams& p, const Unit& un, int j0, int) {
    if (is_gate_up(MODE))
      weight = j0 + static_cast<int>(threadIdx.x & 31) < un.used ? p.plan.row_weight[un.row0 + j0 + (threadIdx.x & 31)] : 0.f;
  }
};
template <>
struct Prefetched<kDHidden> {
  static constexpr int kBatch = 4;
  float weight = 0.f;
  float2 gu[kBatch];  // gate/up products of the first rows; write_rows fetches the others
  // Rows and columns that do not exist are read at the tile's first and not used: no branches.
  __device__ __forceinline__ static void batch(const RowsParams& p, const Unit& un, int j0, int col, float2 (&to)[kBatch]) {
    const float2* src =
        reinterpret_cast<const float2*>(p.gu) + static_cast<long long>(un.row0) * p.cols + (col < p.cols ? col : 0);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      to[j] = __ldcs(src + static_cast<long long>(j0 + j < un.used ? j0 + j : 0) * p.cols);
  }
  __device__ __forceinline__ void fetch(const RowsParams& p, const Unit& un, int j0, int col) {
    const int j = j0 + static_cast<int>(threadIdx.x & 31);
    weight = j < un.used ? p.plan.row_weight[un.row0 + j] : 0.f;
    batch(p, un, j0, col, gu);
  }
};

// Output of 32 rows (from row j0 of the tile) x 32 columns (a lane each), r[j] = product of row j0 + j.
// WHOLE: all rows are in use and all columns exist.
template <int MODE, bool BF16, bool WHOLE>
__device__ __forceinline__ void write_rows(const RowsParams& p, const Unit& un, int j0, int rows, int warp_col, int lane,
                                           uint32_t (&r)[32], Prefetched<MODE>& pre) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const long long row = un.row0 + j0;
  const int col = warp_col + lane;
  const bool inside = WHOLE || col < p.cols;
  const int used = un.used - j0, write = rows - j0;  // of these 32
  if (MODE == kDown || MODE == kDX) {
    float* dst = static_cast<float*>(p.out) + (un.slice * p.max_rows + row) * p.cols + col;
#pragma unroll
    for (int j = 0; j < 32; ++j, dst += p.cols)
      if (WHOLE || (inside && j < write)) *dst = __uint_as_float(r[j]);
  } else if (is_gate_up(MODE)) {
    if (MODE == kGateUpKeep) {
      float* dst = p.gu + row * p.cols + col;
#pragma unroll
      for (int j = 0; j < 32; ++j, dst += p.cols)
        if (WHOLE || (inside && j < used)) *dst = __uint_as_float(r[j]);
    }
    // Even lanes hold gates, odd lanes their up columns.  For four rows at a time: lanes of a pair
    // exchange so that each has both products of one of two rows, then lanes two apart so that each
    // has two neighbouring hidden columns of one row: 4 bytes to store.
    const bool odd = (lane & 1) != 0, second = (lane & 2) != 0;
    const int d_ff = p.cols >> 1, hidden_col = (warp_col >> 1) + (lane >> 2) * 2;
    T* dst = static_cast<T*>(p.out) + (row + (lane & 1) + (lane & 2)) * d_ff + hidden_col;
#pragma unroll
    for (int j = 0; j < 32; j += 4, dst += 4 * d_ff) {
      if (!WHOLE && j >= write) break;
      float z[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int ja = j + 2 * h;
        const float x = __uint_as_float(__shfl_xor_sync(0xffffffffu, odd ? r[ja] : r[ja + 1], 1));
        const float g = odd ? x : __uint_as_float(r[ja]);
        const float up = odd ? __uint_as_float(r[ja + 1]) : x;
        const float w = __shfl_sync(0xffffffffu, pre.weight, ja + (lane & 1));
        z[h] = w * up * gate_act(g, p.activation).x;
        if (!WHOLE && ja + (lane & 1) >= used) z[h] = 0.f;
      }
      const float y = __shfl_xor_sync(0xffffffffu, second ? z[0] : z[1], 2);
      const uint32_t pair = second ? pack2<BF16>(y, z[1]) : pack2<BF16>(z[0], y);
      if (WHOLE || (hidden_col < d_ff && j + (lane & 3) < write)) *reinterpret_cast<uint32_t*>(dst) = pair;
    }
  } else {
    // dG = w dH up act'(gate), dUp = w dH act(gate); dw = sum over hidden columns of dH H
    constexpr int kBatch = Prefetched<kDHidden>::kBatch;
    auto& first = reinterpret_cast<Prefetched<kDHidden>&>(pre);
    uint32_t* dst = static_cast<uint32_t*>(p.out) + row * p.cols + col;
    float2 other[kBatch];
    // (a row's part of dw takes the place of its dH)
#pragma unroll
    for (int b = 0; b < 32; b += 2 * kBatch) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        auto& now = h == 0 ? first.gu : other;
        if (b + h * kBatch + kBatch < 32)
          Prefetched<kDHidden>::batch(p, un, j0 + b + (h + 1) * kBatch, col, h == 0 ? other : first.gu);
#pragma unroll
        for (int i = 0; i < kBatch; ++i, dst += p.cols) {
          const int j = b + h * kBatch + i;
          const float d = __uint_as_float(r[j]);
          const float2 a = gate_act(now[i].x, p.activation);
          const float wd = __shfl_sync(0xffffffffu, first.weight, j) * d;
          r[j] = WHOLE || (inside && j < used) ? __float_as_uint(d * (a.x * now[i].y)) : 0u;
          const uint32_t pair = pack2<BF16>(wd * now[i].y * a.y, wd * a.x);
          if (WHOLE || (inside && j < write)) *dst = WHOLE || j < used ? pair : 0u;
        }
      }
    }
    const float sum = transposed_sum(r, lane);
    if (WHOLE || lane < used) p.dw_part[(row + lane) * p.dw_parts + (warp_col >> 5)] = sum;
  }
}

__device__ __forceinline__ uint32_t add_bits(uint32_t a, uint32_t b) {
  return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}

// out^T[256 columns, n rows] = W^T rows^T for one expert's rows; see the top of the file.
// tmap_w: the weights.  kGateUp, kDown: K runs down their rows, M along them: 64 x 128 boxes, two at
// a time where the columns are whole panels of 64 (p.panels); kDHidden, kDX: M down, K along: 64 x
// 128 boxes, one per slab.  tmap_r: the rows, 64 elements by 128, 64, 32 and 16 rows, so that a copy
// is made of exactly the rows a tile has (kGateUpGather: tmap_r.m[3] is x itself, one row high).
// What bounds these products is the way from L2 to the SMs: 64 KB for 1024 cycles of a full stage's
// MMAs is the 64 bytes per cycle an SM can take at most.
template <int MODE, bool BF16>
__global__ void __launch_bounds__(kRowsThreads, 1)
moe_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ RowsMaps tmap_r,
                const RowsParams p) {
  constexpr bool gate_up = is_gate_up(MODE);
  constexpr bool gather = MODE == kGateUpGather;
  constexpr bool w_kmajor = MODE == kDHidden || MODE == kDX;
  constexpr int kSumBlocks = sum_blocks(BF16);
  constexpr int operand_bytes = kRows * kTileK * 2;
  constexpr int kSlabBytes = kRows * kSlab * 2;       // K-major: 128 rows x 64 elements
  constexpr int kAtom = kTileK * kAtomBytes;          // M-major: 64 columns x K rows
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  const uint32_t smem_w = (raw_addr + 1023u) & ~1023u;
  const uint32_t smem_r = smem_w + p.stages * operand_bytes;
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(smem_raw + (smem_r + p.stages * operand_bytes - raw_addr));
  float* parked = reinterpret_cast<float*>(reinterpret_cast<char*>(ctrl) + kCtrlBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x >> 1;
  const int num_clusters = gridDim.x >> 1;
  volatile int* abort_flag = &ctrl->abort;
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tmap_w);
    for (int i = 0; i < 4; ++i) ptx::prefetch_tensormap(&tmap_r.m[i]);
  }
  const uint32_t tmem_base = set_up_pair(ctrl, p.stages, kRowsEpilogue, warp);
  // Everything above touches no global memory and may run under the tail of the kernel before.
  dependency_wait();
  dependency_release();
  const int num_tiles = *p.plan.tiles;
  const int total_units = num_tiles * p.tiles_n * p.splits;

  if (warp == 0) {
    // ===== TMA producer: every lane issues its share of a stage's copies =====
    Cursor ring;
    bool ok = true;
    for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
      const Unit un = decode_unit<MODE>(p, u, num_tiles);
      const int half = un.n >> 1;  // rows each CTA fetches
      const int row0 = un.row0 + rank * half;
      const int w_col = un.col0 + rank * kRows;
      const int slab_bytes = half * kAtomBytes + (w_kmajor ? kSlabBytes : 0);
      // lanes 0 to 3 copy 128, 64, 32 and 16 rows: the binary digits of `half`, largest first
      const int size = 128 >> (lane & 3);
      const bool copies = lane < 4 && (half & size) != 0;
      const int from = half & ~(2 * size - 1);
      int rows[4] = {0, 0, 0, 0};
      if (gather) {
        // rows past the last are copies of that one: addressable, and never stored
        const int last = un.row0 + un.used - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) rows[i] = p.plan.row_token[min(row0 + 4 * lane + i, last)];
      }
      for (int kb = 0; kb < un.num_kb; ++kb) {
        const bool got = ptx::mbar_wait(ptx::smem_u32(&ctrl->empty[ring.at]), ring.phase ^ 1u, abort_flag, p.timeout_ns);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        const uint32_t full_bar = ptx::smem_u32(&ctrl->full[ring.at]);
        const int k0 = (un.kb0 + kb) * kTileK;
        const int slabs = p.k - k0 > kSlab ? 2 : 1;  // (nothing reads the second slab of a short last block)
        if (leader && lane == 0)
          ptx::mbar_arrive_expect_tx(full_bar, 2u * static_cast<uint32_t>(slabs * slab_bytes + (w_kmajor ? 0 : operand_bytes)));
        const uint32_t bar = ptx::mapa(full_bar, 0);  // both CTAs' copies complete on the leader's barrier
        __syncwarp();
        const uint32_t w_dst = smem_w + ring.at * operand_bytes;
        const uint32_t r_dst = smem_r + ring.at * operand_bytes;
        if (!w_kmajor && p.panels) {
          if (lane == 31) ptx::tma_load_4d_pair(w_dst, &tmap_w, 0, k0, w_col >> 6, un.expert, bar);
        } else if (!w_kmajor && lane >= 30) {
          const int half_w = lane - 30;
          ptx::tma_load_3d_pair(w_dst + half_w * kAtom, &tmap_w, w_col + half_w * 64, k0, un.expert, bar);
        }
        for (int slab = 0; slab < slabs; ++slab) {
          const int k = k0 + slab * kSlab;
          const uint32_t dst = r_dst + slab * kSlabBytes;
          if (w_kmajor && lane == 31)
            ptx::tma_load_3d_pair(w_dst + slab * kSlabBytes, &tmap_w, k, w_col, un.expert, bar);
          if (gather) {
            if (4 * lane < half) tma_gather4_pair(dst + lane * 512, &tmap_r.m[3], k, rows, bar);
          } else if (copies) {
            ptx::tma_load_2d_pair(dst + from * kAtomBytes, &tmap_r.m[lane], k, row0 + from, bar);
          }
        }
        __syncwarp();
        ring.next(p.stages);
      }
    }
    if (!ok && lane == 0 && p.status != nullptr) atomicCAS(p.status, 0, kAbortProducer);
  } else if (warp == 1) {
    // ===== MMA issuer (leader CTA) =====
    if (leader && lane == 0) {
      const uint32_t fmt = BF16 ? 1u : 0u;
      // fp32 accumulate, M = 256 weight columns, N = the tile's rows (K-major)
      const uint32_t idesc_base = (1u << 4) | (fmt << 7) | (fmt << 10) | ((w_kmajor ? 0u : 1u) << 15) |
                                  (static_cast<uint32_t>((kRows * 2) >> 4) << 24);
      // K-major operands: slabs of 128 rows x 128 bytes, 16 elements of K = 32 bytes further.  An
      // M-major one: 64-wide atoms of 128 K rows x 128 bytes, 16 elements of K = 16 rows.
      const uint64_t w_desc =
          w_kmajor ? ptx::make_smem_desc(0, 0, 1024) : ptx::make_smem_desc(0, kAtom, 1024);
      const uint64_t r_desc = ptx::make_smem_desc(0, 0, 1024);
      Cursor ring, acc;
      bool ok = true;
      for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
        const Unit un = decode_unit<MODE>(p, u, num_tiles);
        const uint32_t idesc = idesc_base | (static_cast<uint32_t>(un.n >> 3) << 17);
        uint32_t d_tmem = 0, accumulate = 0;
        for (int kb = 0; kb < un.num_kb; ++kb) {
          if (kb == 0 || (sums_outside(MODE) && kb % kSumBlocks == 0)) {  // a fresh accumulator
            if (!ptx::mbar_wait<true>(ptx::smem_u32(&ctrl->tmem_empty[acc.at]), acc.phase ^ 1u, abort_flag,
                                      p.timeout_ns)) {
              ok = false;
              break;
            }
            ptx::tc_fence_after_sync();
            d_tmem = tmem_base + acc.at * kTileN;
            accumulate = 0;
          }
          if (!ptx::mbar_wait(ptx::smem_u32(&ctrl->full[ring.at]), ring.phase, abort_flag, p.timeout_ns)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t w16 = (smem_w + ring.at * operand_bytes) >> 4;
          const uint32_t r16 = (smem_r + ring.at * operand_bytes) >> 4;
          const int steps = (p.k - (un.kb0 + kb) * kTileK + 15) >> 4;
#pragma unroll
          for (int k16 = 0; k16 < kTileK / 16; ++k16) {
            const uint32_t in_slab = (k16 & 3) * 2u;
            const uint32_t w_off = w_kmajor ? (k16 >> 2) * (kSlabBytes >> 4) + in_slab : k16 * 128u;
            const uint32_t r_off = (k16 >> 2) * (kSlabBytes >> 4) + in_slab;
            if (k16 < steps)
              ptx::umma_f16<2>(d_tmem, w_desc | ((w16 + w_off) & 0x3fffu), r_desc | ((r16 + r_off) & 0x3fffu), idesc,
                               accumulate);
            accumulate = 1;
          }
          ptx::umma_commit_pair(ptx::smem_u32(&ctrl->empty[ring.at]), 0x3);
          ring.next(p.stages);
          if (kb + 1 == un.num_kb || (sums_outside(MODE) && (kb + 1) % kSumBlocks == 0)) {
            ptx::umma_commit_pair(ptx::smem_u32(&ctrl->tmem_full[acc.at]), 0x3);
            acc.next(2);
          }
        }
      }
      if (!ok && p.status != nullptr) atomicCAS(p.status, 0, kAbortMma);
    }
  } else {
    // ===== epilogue: warp w owns TMEM lanes 32 (w mod 4) ..., i.e. 32 columns of the output; a
    // register is a row.  Four warps share the columns and take every fourth 32 rows.  A warp's
    // arithmetic is one dependent chain after another (about 7 cycles per instruction were
    // measured), so it takes this many warps to stay ahead of the products: with four (eight)
    // the gate/up product of 8192 tokens, 64 experts 2048/1024 took 523 (449) us. =====
    const int quarter = warp & 3;
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const int first_row = ((warp - 2) >> 2) * 32;
    constexpr int kStep = 8 * kRowsEpilogue;  // rows from one of a warp's chunks to its next
    Cursor acc;
    bool ok = true;
    for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
      const Unit un = decode_unit<MODE>(p, u, num_tiles);
      const int warp_col = un.col0 + rank * kRows + quarter * 32;
      // rows to write: those in use, and in a training step the zeros that pad an expert (products
      // over K = rows read them)
      const int rows = sums_outside(MODE) ? un.padded : un.used;
      const int mine = warp_col < p.cols ? rows : 0;  // (warp-uniform)
      Prefetched<MODE> pre;
      // Waits for the next accumulator; false if it does not come in time.
      auto next_accumulator = [&]() -> bool {
        const bool got = ptx::mbar_wait(ptx::smem_u32(&ctrl->tmem_full[acc.at]), acc.phase, abort_flag, p.timeout_ns);
        if (!__all_sync(0xffffffffu, got)) return false;
        ptx::tc_fence_after_sync();
        return true;
      };
      uint32_t r[32];
      auto write = [&](int j0) {
        if (j0 + 32 <= un.used && warp_col + 32 <= p.cols)
          write_rows<MODE, BF16, true>(p, un, j0, rows, warp_col, lane, r, pre);
        else
          write_rows<MODE, BF16, false>(p, un, j0, rows, warp_col, lane, r, pre);
      };
      if constexpr (sums_outside(MODE)) {
        // The sums over kSumBlocks K blocks each, added in fp32 as they come: the first 32 rows and
        // half of the second in registers, the other half in this thread's column of `parked`.
        static_assert(kTileN == 2 * kStep, "a warp has two chunks of rows");
        float* mine_parked = parked + (warp - 2) * (kParkedRows * 32) + lane;
        const bool one = first_row < mine, two = first_row + kStep < mine;
        uint32_t more[32 - kParkedRows];
        const int parts = (un.num_kb + kSumBlocks - 1) / kSumBlocks;
        for (int part = 0; part < parts; ++part) {
          if (!next_accumulator()) {
            ok = false;
            break;
          }
          const uint32_t t_acc = tmem_base + lane_sel + acc.at * kTileN + first_row;
          if (one) {
            uint32_t v[16];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ptx::tmem_ld_32x16(t_acc + half * 16, v);
              ptx::tmem_ld_wait(v);
#pragma unroll
              for (int j = 0; j < 16; ++j) r[half * 16 + j] = part == 0 ? v[j] : add_bits(r[half * 16 + j], v[j]);
            }
            if (two) {
              ptx::tmem_ld_32x16(t_acc + kStep, v);
              ptx::tmem_ld_wait(v);
#pragma unroll
              for (int j = 0; j < 16; ++j) more[j] = part == 0 ? v[j] : add_bits(more[j], v[j]);
              ptx::tmem_ld_32x16(t_acc + kStep + 16, v);
              ptx::tmem_ld_wait(v);
              release_accumulator(ctrl, acc.at, leader, lane);
#pragma unroll
              for (int j = 0; j < 16; ++j)
                mine_parked[j * 32] = (part == 0 ? 0.f : mine_parked[j * 32]) + __uint_as_float(v[j]);
            }
          }
          if (!two) release_accumulator(ctrl, acc.at, leader, lane);
          acc.next(2);
        }
        if (!ok) break;
        if (one) {
          pre.fetch(p, un, first_row, warp_col + lane);
          write(first_row);
        }
        if (two) {
          pre.fetch(p, un, first_row + kStep, warp_col + lane);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            r[j] = more[j];
            r[16 + j] = __float_as_uint(mine_parked[j * 32]);
          }
          write(first_row + kStep);
        }
      } else {
        if (first_row < mine) pre.fetch(p, un, first_row, warp_col + lane);
        if (!next_accumulator()) {
          ok = false;
          break;
        }
        const uint32_t t_acc = tmem_base + lane_sel + acc.at * kTileN;
        for (int j0 = first_row; j0 < mine; j0 += kStep) {
          ptx::tmem_ld_32x32(t_acc + j0, r);
          ptx::tmem_ld_wait(r);
          write(j0);
          if (j0 + kStep < mine) pre.fetch(p, un, j0 + kStep, warp_col + lane);
        }
        release_accumulator(ctrl, acc.at, leader, lane);
        acc.next(2);
      }
    }
    if (!ok && lane == 0 && p.status != nullptr) atomicCAS(p.status, 0, kAbortEpilogue);
  }
  tear_down_pair(ctrl, tmem_base, warp);
}

// out[e] (m x n) = A[rows of e]^T B[rows of e]: tmap_a and tmap_b are 64 x 128 boxes over matrices of
// rows in expert order, tmap_c 64 x 32 boxes over the gradients.  An expert's last K block ends at
// the padding (zeros in both operands): one to eight MMAs of 16 rows.
template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
moe_wgrad_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                 const __grid_constant__ CUtensorMap tmap_c, const WgradParams p) {
  constexpr int operand_bytes = kRows * kTileK * 2;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  const uint32_t smem_a = (raw_addr + 1023u) & ~1023u;
  const uint32_t smem_b = smem_a + p.stages * operand_bytes;
  const uint32_t smem_out = smem_b + p.stages * operand_bytes;
  Ctrl* ctrl = reinterpret_cast<Ctrl*>(smem_raw + (smem_out + 4 * kBoxes * kBoxBytes - raw_addr));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = static_cast<int>(ptx::cluster_ctarank());
  const bool leader = rank == 0;
  const int cluster_id = blockIdx.x >> 1;
  const int num_clusters = gridDim.x >> 1;
  volatile int* abort_flag = &ctrl->abort;
  if (threadIdx.x == 0) {
    ptx::prefetch_tensormap(&tmap_a);
    ptx::prefetch_tensormap(&tmap_b);
    ptx::prefetch_tensormap(&tmap_c);
  }
  const uint32_t tmem_base = set_up_pair(ctrl, p.stages, 4, warp);
  dependency_wait();
  dependency_release();
  const int per_expert = p.tiles_m * p.tiles_n;
  const int total_units = p.experts * per_expert;

  if (warp == 0) {
    Cursor ring;
    bool ok = true;
    for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
      const int e = u / per_expert, rem = u - e * per_expert, tn = rem / p.tiles_m;
      const int m0 = (rem - tn * p.tiles_m) * (2 * kRows) + rank * kRows;
      const int n0 = tn * kTileN + rank * kRows;
      const int k_row0 = p.plan.start[e], num_kb = (p.plan.count[e] + kTileK - 1) / kTileK;
      for (int kb = 0; kb < num_kb; ++kb) {
        const bool got = ptx::mbar_wait(ptx::smem_u32(&ctrl->empty[ring.at]), ring.phase ^ 1u, abort_flag, p.timeout_ns);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        const uint32_t full_bar = ptx::smem_u32(&ctrl->full[ring.at]);
        if (leader && lane == 0) ptx::mbar_arrive_expect_tx(full_bar, 4u * operand_bytes);
        const uint32_t bar = ptx::mapa(full_bar, 0);
        __syncwarp();
        const int k = k_row0 + kb * kTileK;
        const uint32_t a_dst = smem_a + ring.at * operand_bytes, b_dst = smem_b + ring.at * operand_bytes;
        if (p.panels_a) {
          if (lane == 0) ptx::tma_load_4d_pair(a_dst, &tmap_a, 0, k, m0 >> 6, 0, bar);
        } else if (lane < 2) {
          ptx::tma_load_2d_pair(a_dst + lane * (operand_bytes / 2), &tmap_a, m0 + lane * 64, k, bar);
        }
        if (p.panels_b) {
          if (lane == 2) ptx::tma_load_4d_pair(b_dst, &tmap_b, 0, k, n0 >> 6, 0, bar);
        } else if (lane == 2 || lane == 3) {
          ptx::tma_load_2d_pair(b_dst + (lane - 2) * (operand_bytes / 2), &tmap_b, n0 + (lane - 2) * 64, k, bar);
        }
        __syncwarp();
        ring.next(p.stages);
      }
    }
    if (!ok && lane == 0 && p.status != nullptr) atomicCAS(p.status, 0, kAbortProducer);
  } else if (warp == 1) {
    if (leader && lane == 0) {
      const uint32_t fmt = BF16 ? 1u : 0u;
      // fp32 accumulate, both operands MN-major, 256 x 256
      const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 15) | (1u << 16) |
                             (static_cast<uint32_t>(kTileN >> 3) << 17) | (static_cast<uint32_t>((kRows * 2) >> 4) << 24);
      const uint64_t desc = ptx::make_smem_desc(0, operand_bytes / 2, 1024);
      Cursor ring, acc;
      bool ok = true;
      for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
        const int count = p.plan.count[u / per_expert];
        const int num_kb = (count + kTileK - 1) / kTileK;
        if (num_kb == 0) continue;  // an expert without rows: the epilogue writes zeros by itself
        if (!ptx::mbar_wait<true>(ptx::smem_u32(&ctrl->tmem_empty[acc.at]), acc.phase ^ 1u, abort_flag, p.timeout_ns)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc.at * kTileN;
        uint32_t accumulate = 0;
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!ptx::mbar_wait(ptx::smem_u32(&ctrl->full[ring.at]), ring.phase, abort_flag, p.timeout_ns)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after_sync();
          const uint32_t a16 = (smem_a + ring.at * operand_bytes) >> 4;
          const uint32_t b16 = (smem_b + ring.at * operand_bytes) >> 4;
          const int steps = min(kTileK / 16, (count - kb * kTileK + 15) / 16);
#pragma unroll
          for (int k16 = 0; k16 < kTileK / 16; ++k16) {
            if (k16 < steps)
              ptx::umma_f16<2>(d_tmem, desc | ((a16 + k16 * 128u) & 0x3fffu), desc | ((b16 + k16 * 128u) & 0x3fffu),
                               idesc, accumulate);
            accumulate = 1;
          }
          ptx::umma_commit_pair(ptx::smem_u32(&ctrl->empty[ring.at]), 0x3);
          ring.next(p.stages);
        }
        if (!ok) break;
        ptx::umma_commit_pair(ptx::smem_u32(&ctrl->tmem_full[acc.at]), 0x3);
        acc.next(2);
      }
      if (!ok && p.status != nullptr) atomicCAS(p.status, 0, kAbortMma);
    }
  } else {
    // a thread owns a row of the tile, a warp stages boxes of 32 rows x 64 columns and stores them
    const int quarter = warp & 3;
    const uint32_t lane_sel = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t my_smem = smem_out + quarter * (kBoxes * kBoxBytes);
    const uint32_t stage_row = static_cast<uint32_t>(lane) * kAtomBytes;
    const uint32_t sw = static_cast<uint32_t>(lane & 7);
    Cursor acc;
    uint32_t stores = 0;
    bool ok = true;
    for (int u = cluster_id; u < total_units && ok; u += num_clusters) {
      const int e = u / per_expert, rem = u - e * per_expert, tn = rem / p.tiles_m;
      const int row0 = (rem - tn * p.tiles_m) * (2 * kRows) + rank * kRows + quarter * 32;
      const int n0 = tn * kTileN;
      const bool empty = p.plan.count[e] == 0;
      if (!empty) {
        const bool got = ptx::mbar_wait(ptx::smem_u32(&ctrl->tmem_full[acc.at]), acc.phase, abort_flag, p.timeout_ns);
        if (!__all_sync(0xffffffffu, got)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after_sync();
      }
      const uint32_t t_acc = tmem_base + lane_sel + acc.at * kTileN;
      for (int c = 0; c < kTileN && row0 < p.m && n0 + c < p.n; c += 64) {
        // a box that no store reads any more
        if (lane == 0) ptx::tma_store_wait_read<kBoxes - 1>();
        __syncwarp();
        const uint32_t buf = my_smem + (stores++ % kBoxes) * kBoxBytes;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
          uint32_t r[32];
          if (!empty) {
            ptx::tmem_ld_32x32(t_acc + c + sub * 32, r);
            ptx::tmem_ld_wait(r);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = 0u;
          }
#pragma unroll
          for (uint32_t piece = 0; piece < 4; ++piece)
            st_shared_v4(buf + stage_row + ((sub * 4 + piece) ^ sw) * 16,
                         pack2<BF16>(__uint_as_float(r[piece * 8]), __uint_as_float(r[piece * 8 + 1])),
                         pack2<BF16>(__uint_as_float(r[piece * 8 + 2]), __uint_as_float(r[piece * 8 + 3])),
                         pack2<BF16>(__uint_as_float(r[piece * 8 + 4]), __uint_as_float(r[piece * 8 + 5])),
                         pack2<BF16>(__uint_as_float(r[piece * 8 + 6]), __uint_as_float(r[piece * 8 + 7])));
        }
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          ptx::tma_store_3d(&tmap_c, n0 + c, row0, e, buf);
          ptx::tma_store_commit();
        }
      }
      if (!empty) {
        release_accumulator(ctrl, acc.at, leader, lane);
        acc.next(2);
      }
    }
    if (lane == 0) ptx::tma_store_wait_all<0>();
    if (!ok && lane == 0 && p.status != nullptr) atomicCAS(p.status, 0, kAbortEpilogue);
  }
  tear_down_pair(ctrl, tmem_base, warp);
}

// ----------------------------------------------------------------------- rows in and out of order

// out[pos[t, s]] = in[t] for every slot: a 16-byte piece of a token is read once and stored top_k
// times.  The blocks from `copy_blocks` on (where there are any) clear an expert's padding rows each,
// which products over K = rows read.
__global__ void __launch_bounds__(256) permute_kernel(const Plan plan, const uint4* in, long long ld_in, uint4* out,
                                                      int tokens, int top_k, int vectors, int copy_blocks) {
  dependency_wait();
  dependency_release();
  if (static_cast<int>(blockIdx.x) >= copy_blocks) {
    const int e = blockIdx.x - copy_blocks;
    const int count = plan.count[e];
    const long long first = static_cast<long long>(plan.start[e] + count) * vectors;
    const int clear = ((count + kPad - 1) / kPad * kPad - count) * vectors;
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

// out[t] = sum over slots and slices of part[slice][pos[t, s]], in order; slots without an expert
// add nothing.
template <typename T>
__global__ void __launch_bounds__(256) combine_kernel(const float* part, const int* pos, T* out, long long ld_out,
                                                      int tokens, int top_k, int cols, int splits,
                                                      long long slice) {
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
      for (int q = 0; q < splits; ++q) {
        float v[8];
        elem::load<float, 8>(part + q * slice + static_cast<long long>(row) * cols + c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += v[j];
      }
    }
    elem::store<T, 8>(out + t * ld_out + c, sum);
  }
}

// dweights[pair] = sum over the parts of the pair's row: 16 lanes per pair, each adding every
// sixteenth part, then pairwise.
__global__ void __launch_bounds__(256) weight_grad_kernel(const float* dw_part, const int* pos, float* dweights,
                                                          int pairs, int parts) {
  dependency_wait();
  dependency_release();
  const int i = blockIdx.x * 16 + (threadIdx.x >> 4), lane = threadIdx.x & 15;
  const int row = i < pairs ? pos[i] : -1;
  float sum = 0.f;
  if (row >= 0)
    for (int c = lane; c < parts; c += 16) sum += dw_part[static_cast<long long>(row) * parts + c];
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (i < pairs && lane == 0) dweights[i] = sum;
}

// ------------------------------------------------------------------------------------ one token
//
// For a single token every expert's weights are read for one row, and reading them is all there is
// to do: 100 MB for 8 experts of 2048/1024, 15.6 us at the measured copy rate.  stream_kernel reads
// them with 16-byte loads, eight to sixteen rows of weights per warp in flight, and multiplies on
// the CUDA cores in fp32: a block owns one expert, 256 columns and a slice of K.  The slices fill
// the SMs three blocks deep; their sums meet in fp32 in the next kernel, in order: the gate/up
// slices when the down product computes its hidden activation (which is never rounded here), the
// down slices in stream_join_kernel.  No sorting, no row tiles.  (From two tokens on the tiles win:
// rows that share an expert would have to share a read, and four rows at a time the CUDA cores
// bound this kernel: 2 tokens 82 us, 4 tokens 111 us against 86 us for 5 tokens in tiles.)
constexpr int kStreamPairs = 32;
constexpr int kStreamThreads = 256;
constexpr int kStreamCols = 256;   // a warp's 32 lanes x 8 columns
constexpr int kStreamMaxK = 1024;  // of a slice

struct StreamParams {
  const void* ids;
  int wide, experts, pairs, top_k;
  const float* weights;
  const void* x;       // gate/up: rows of x
  long long ld_x;
  const float* parts;  // down: gate/up sums, [pairs][parts_n][2 k]
  int parts_n;
  const void* w;       // weights [experts][k][cols]
  long long expert_pitch, row_pitch;
  int k, cols, slices, slice_k;  // slice_k: a multiple of 64
  int activation;
  float* out;          // [pairs][slices][cols]
};

__device__ __forceinline__ uint4 load_streaming(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <typename T, bool DOWN>
__global__ void __launch_bounds__(kStreamThreads, 3) stream_kernel(const StreamParams p) {
  __shared__ float row[kStreamMaxK];  // this slice of a pair's row
  __shared__ float sums[8][kStreamCols + 8];
  __shared__ int list[kStreamPairs];
  __shared__ int list_n;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int slice = blockIdx.x % p.slices, chunk = blockIdx.x / p.slices;
  const int k0 = slice * p.slice_k, k1 = min(k0 + p.slice_k, p.k);
  const int col = chunk * kStreamCols + lane * 8;
  // (ids and weights were complete before the kernel ahead of this one started: see
  // dependency_release() there)
  if (!DOWN) {
    dependency_wait();
    dependency_release();
  }
  const int pair = blockIdx.y;
  const int e = pair_expert(p.ids, p.wide, p.experts, pair);
  // the first pair of an expert works for all of them
  if (warp == 0) {
    int n = 0;
    bool first = e >= 0;
    for (int base = 0; base < p.pairs; base += 32) {
      const int i = base + lane;
      const bool same = i < p.pairs && e >= 0 && pair_expert(p.ids, p.wide, p.experts, i) == e;
      const unsigned mask = __ballot_sync(0xffffffffu, same);
      if (__ballot_sync(0xffffffffu, same && i < pair) != 0) first = false;
      if (same) list[n + __popc(mask & ((1u << lane) - 1u))] = i;
      n += __popc(mask);
    }
    if (lane == 0) list_n = first ? n : 0;
  }
  const T* w = static_cast<const T*>(p.w) + static_cast<long long>(e < 0 ? 0 : e) * p.expert_pitch + col;
  const bool inside = col < p.cols;
  // A warp's rows of weights: k0 + 8 warp + 64 i + (0..7).  The first eight are on their way before
  // anything this kernel depends on is waited for.
  uint4 v[8];
  auto fetch = [&](int k) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = inside && k + j < k1 ? load_streaming(w + static_cast<long long>(k + j) * p.row_pitch) : make_uint4(0, 0, 0, 0);
  };
  __syncthreads();
  const int n = list_n;
  if (n > 0) fetch(k0 + warp * 8);
  if (DOWN) {
    dependency_wait();
    dependency_release();
  }
  for (int r = 0; r < n; ++r) {  // (more than one only where an expert stands in several slots)
    const int q = list[r];
    for (int i = tid; i < p.slice_k; i += kStreamThreads) {
      const int k = k0 + i;
      float val = 0.f;
      if (k < k1) {
        if (DOWN) {
          const float2* src = reinterpret_cast<const float2*>(p.parts) + static_cast<long long>(q) * p.parts_n * p.k + k;
          float2 gu = make_float2(0.f, 0.f);
#pragma unroll 8
          for (int s = 0; s < p.parts_n; ++s) {
            const float2 part = src[static_cast<long long>(s) * p.k];
            gu.x += part.x;
            gu.y += part.y;
          }
          val = p.weights[q] * gate_act(gu.x, p.activation).x * gu.y;
        } else {
          val = elem::to_float(static_cast<const T*>(p.x)[q / p.top_k * p.ld_x + k]);
        }
      }
      row[i] = val;
    }
    __syncthreads();
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (r > 0) fetch(k0 + warp * 8);
    for (int i = warp * 8; i < p.slice_k; i += 64) {
      uint4 now[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) now[j] = v[j];
      if (i + 64 < p.slice_k) fetch(k0 + i + 64);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const T* t = reinterpret_cast<const T*>(&now[j]);
        const float a = row[i + j];
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[c] += a * elem::to_float(t[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < 8; c += 4)
      *reinterpret_cast<float4*>(&sums[warp][lane * 8 + c]) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    __syncthreads();
    const int c = chunk * kStreamCols + tid;
    if (c < p.cols) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += sums[i][tid];
      p.out[(static_cast<long long>(q) * p.slices + slice) * p.cols + c] = sum;
    }
    // (the next round's writes of `row` and `sums` are a barrier away from this one's reads)
    __syncthreads();
  }
}

// y[t] = sum over slots and slices, in order within each of eight strands, then pairwise.
template <typename T>
__global__ void __launch_bounds__(256) stream_join_kernel(const StreamParams p, T* y, long long ld_y) {
  __shared__ float sums[8][33];
  const int c = blockIdx.x * 32 + threadIdx.x, strand = threadIdx.y, t = blockIdx.y;
  dependency_wait();
  dependency_release();
  float sum = 0.f;
  if (c < p.cols)
#pragma unroll 8
    for (int i = strand; i < p.top_k * p.slices; i += 8) {
      const int q = t * p.top_k + i / p.slices;
      if (pair_expert(p.ids, p.wide, p.experts, q) >= 0)
        sum += p.out[(static_cast<long long>(q) * p.slices + i % p.slices) * p.cols + c];
    }
  sums[strand][threadIdx.x] = sum;
  __syncthreads();
  if (strand == 0 && c < p.cols) {
    for (int i = 1; i < 8; ++i) sum += sums[i][threadIdx.x];
    y[t * ld_y + c] = elem::from_float<T>(sum);
  }
}

// ------------------------------------------------------------------------------------- host

inline int cdiv(int a, int b) { return (a + b - 1) / b; }
inline int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// Sizes and offsets of one problem.
struct Layout {
  int pairs, max_tiles;
  int64_t max_rows;
  int chunk, chunks;
  bool gather;                 // the copy engine picks the rows of x
  bool stream;                 // one token: stream_kernel
  int up_slices, up_slice_k, down_slices, down_slice_k;
  int64_t up_bytes, down_bytes;
  int down_splits, dx_splits;  // slices of K of the two products with fp32 rows
  int dw_parts;
  // The plan, the hidden activation and the gate/up products: in `saved` when training.
  int64_t off_tiles, off_count, off_start, off_tile, off_row_token, off_row_weight, off_pos, plan_bytes;
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
  // (tile numbers are 32-bit, with up to eight slices of K per tile)
  const int64_t row_tiles = static_cast<int64_t>(p->tokens) * p->top_k / kTileN + p->experts;
  int64_t widest = p->d_model > 2 * p->d_ff ? p->d_model : 2 * p->d_ff;
  if (widest < p->n_out) widest = p->n_out;
  const int64_t col_tiles = widest / 256 + 1, weight_tiles = p->experts * col_tiles;
  if ((row_tiles > weight_tiles ? row_tiles : weight_tiles) * col_tiles > (1 << 27)) {
    set_error("problem has too many tiles");
    return TNX_ERR_INVALID;
  }
  return TNX_OK;
}

// Slices of K for a product with `cols` output columns over num_kb K blocks: the number that takes
// the least time when a K block costs 0.6 us, a tile 2 us of its own, and each slice writes and
// reads its copy of the rows at 6 TB/s.  With few tiles this fills the last wave (8 experts of
// 4096/14336, 500 tokens: 128 tiles for 74 pairs of SMs).
int pick_splits(const Layout& l, int cols, int num_kb) {
  const int clusters = sm_count() / 2;
  const double units = static_cast<double>(l.max_tiles) * cdiv(cols, 2 * kRows);
  int best = 1;
  double least = 0.0;
  for (int s = 1; s <= 8 && num_kb / s >= 2; s *= 2) {
    const int waves = static_cast<int>((units * s + clusters - 1) / clusters);
    const double us = waves * (0.6 * cdiv(num_kb, s) + 2.0) + s * (8.0 * l.pairs * cols / 6.0e6);
    if (s == 1 || us < 0.95 * least) {
      best = s;
      least = us;
    }
  }
  return best;
}

// Slices of K of the streamed products: three blocks for every SM, slices of 64 to kStreamMaxK.
void pick_slices(int pairs, int cols, int k, int* slices, int* slice_k) {
  const int blocks = pairs * cdiv(cols, kStreamCols);
  int n = cdiv(3 * sm_count(), blocks);
  if (n > cdiv(k, 64)) n = cdiv(k, 64);
  if (n < cdiv(k, kStreamMaxK)) n = cdiv(k, kStreamMaxK);
  *slice_k = cdiv(cdiv(k, n), 64) * 64;
  *slices = cdiv(k, *slice_k);
}

Layout lay_out_problem(const tnx_moe_problem& p) {
  Layout l = {};
  l.pairs = p.tokens * p.top_k;
  l.stream = !p.train && p.tokens == 1 && l.pairs <= kStreamPairs;
  if (l.stream) {
    pick_slices(l.pairs, 2 * p.d_ff, p.d_model, &l.up_slices, &l.up_slice_k);
    pick_slices(l.pairs, p.n_out, p.d_ff, &l.down_slices, &l.down_slice_k);
    l.up_bytes = align256(static_cast<int64_t>(l.pairs) * l.up_slices * p.d_ff * 8);
    l.down_bytes = align256(static_cast<int64_t>(l.pairs) * l.down_slices * p.n_out * 4);
  }
  const int hit = l.pairs < p.experts ? l.pairs : p.experts;  // experts with rows at most
  l.max_tiles = (l.pairs - hit) / kTileN + hit;
  l.max_rows = (static_cast<int64_t>(l.pairs) + static_cast<int64_t>(hit) * (kPad - 1)) / kPad * kPad;
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
  l.off_tile = take(16ll * l.max_tiles);
  l.off_row_token = take(4 * l.max_rows);
  l.off_row_weight = take(4 * l.max_rows);
  l.off_pos = take(4ll * l.pairs);
  l.plan_bytes = at;
  // (a training step needs the rows in order for the weights' gradients anyway)
  l.gather = !p.train && l.pairs / p.experts <= 32;
  l.down_splits = pick_splits(l, p.n_out, cdiv(p.d_ff, kTileK));
  l.dx_splits = pick_splits(l, p.d_model, cdiv(2 * p.d_ff, kTileK));
  l.dw_parts = cdiv(p.d_ff, 32);
  l.x_bytes = l.gather ? 0 : align256(l.max_rows * p.d_model * 2);
  l.dy_bytes = align256(l.max_rows * p.n_out * 2);
  l.hidden_bytes = align256(l.max_rows * p.d_ff * 2);
  l.gu_bytes = align256(l.max_rows * p.d_ff * 8);
  l.part_bytes = align256(l.down_splits * l.max_rows * p.n_out * 4);
  l.dgu_bytes = align256(l.max_rows * p.d_ff * 4);
  l.dx_bytes = align256(l.dx_splits * l.max_rows * p.d_model * 4);
  l.dw_bytes = align256(l.max_rows * l.dw_parts * 4);
  return l;
}

Plan plan_at(const Layout& l, void* base) {
  char* b = static_cast<char*>(base);
  Plan q;
  q.tiles = reinterpret_cast<int*>(b + l.off_tiles);
  q.count = reinterpret_cast<int*>(b + l.off_count);
  q.start = reinterpret_cast<int*>(b + l.off_start);
  q.tile = reinterpret_cast<int4*>(b + l.off_tile);
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
int launch(const char* what, void (*fn)(KArgs...), dim3 grid, dim3 block, int smem, int cluster, cudaStream_t stream,
           Args... args) {
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = block;
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

// One pair of CTAs per pair of SMs, or per unit where there are fewer.
template <typename Fn, typename Params, typename... Maps>
int launch_pairs(Fn fn, int threads, Params p, int staging_bytes, int64_t units, cudaStream_t stream,
                 const Maps&... maps) {
  const int fixed = staging_bytes + kCtrlBytes + kAlignSlack;
  const int fit = (kMaxDynamicSmem - fixed) / kStageBytes;
  p.stages = fit > kMaxStages ? kMaxStages : fit;
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(fn), kMaxDynamicSmem);
  if (e != cudaSuccess) return cuda_failed("experts' products: shared memory", e);
  const int most = sm_count() / 2;
  const int clusters = units < most ? static_cast<int>(units) : most;
  return launch("experts' products", fn, clusters * 2, threads, p.stages * kStageBytes + fixed, 2, stream, maps..., p);
}
// Tensor maps over rows in expert order, as moe_rows_kernel reads them.
int rows_maps(RowsMaps* maps, const void* rows, int dtype, int cols, int64_t max_rows) {
  int rc = TNX_OK;
  for (int i = 0; i < 4 && rc == TNX_OK; ++i)
    rc = make_tmap_2d(&maps->m[i], rows, dtype, cols, max_rows, cols, 64, 128 >> i, true);
  return rc;
}
// A map over the weights [experts][rows][cols] with K down their rows.
int weights_map(CUtensorMap* w, RowsParams* g, const tnx_moe_problem& p, const void* ptr, int cols, int rows,
                int64_t row_pitch, int64_t expert_pitch) {
  g->panels = cols % 64 == 0;
  return g->panels ? make_tmap_panels(w, ptr, p.dtype, cols, rows, p.experts, row_pitch, expert_pitch, kTileK)
                   : make_tmap_3d(w, ptr, p.dtype, cols, rows, p.experts, row_pitch, expert_pitch, 64, kTileK, true);
}
template <int MODE>
int launch_rows(const tnx_moe_problem& q, const Layout& l, const CUtensorMap& w, const RowsMaps& r, RowsParams p,
                cudaStream_t stream) {
  p.tiles_n = cdiv(p.cols, 2 * kRows);
  p.max_rows = l.max_rows;
  p.band = 8;
  const int64_t units = static_cast<int64_t>(l.max_tiles) * p.tiles_n * p.splits;
  constexpr int staging = sums_outside(MODE) ? kRowsEpilogue * kParkedRows * 32 * 4 : 0;
  return q.dtype == TNX_BF16
             ? launch_pairs(moe_rows_kernel<MODE, true>, kRowsThreads, p, staging, units, stream, w, r)
             : launch_pairs(moe_rows_kernel<MODE, false>, kRowsThreads, p, staging, units, stream, w, r);
}
// out[e] = a[rows of e]^T b[rows of e], m x n.
int run_wgrad(const tnx_moe_problem& q, const Layout& l, const Plan& plan, const void* a, int m, const void* b, int n,
              void* out, int32_t* status, cudaStream_t stream) {
  WgradParams p = {};
  p.plan = plan;
  p.experts = q.experts;
  p.m = m;
  p.n = n;
  p.tiles_m = cdiv(m, 2 * kRows);
  p.tiles_n = cdiv(n, kTileN);
  p.status = status;
  p.timeout_ns = bounded_wait_limit_ns();
  CUtensorMap ta, tb, tc;
  p.panels_a = m % 64 == 0;
  p.panels_b = n % 64 == 0;
  auto operand = [&](CUtensorMap* map, const void* ptr, int cols, int panels) {
    return panels ? make_tmap_panels(map, ptr, q.dtype, cols, l.max_rows, 1, cols, l.max_rows * cols, kTileK)
                  : make_tmap_2d(map, ptr, q.dtype, cols, l.max_rows, cols, 64, kTileK, true);
  };
  int rc = operand(&ta, a, m, p.panels_a);
  if (rc == TNX_OK) rc = operand(&tb, b, n, p.panels_b);
  if (rc == TNX_OK)
    rc = make_tmap_3d(&tc, out, q.dtype, n, m, q.experts, n, static_cast<int64_t>(m) * n, 64, 32, false);
  if (rc != TNX_OK) return rc;
  const int64_t units = static_cast<int64_t>(q.experts) * p.tiles_m * p.tiles_n;
  const int staging = 4 * kBoxes * kBoxBytes;
  return q.dtype == TNX_BF16 ? launch_pairs(moe_wgrad_kernel<true>, kThreads, p, staging, units, stream, ta, tb, tc)
                             : launch_pairs(moe_wgrad_kernel<false>, kThreads, p, staging, units, stream, ta, tb, tc);
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
                int cols, int splits, int64_t max_rows, cudaStream_t stream) {
  const long long slice = max_rows * cols;
  const int64_t blocks = (static_cast<int64_t>(tokens) * (cols / 8) + 255) / 256;
  const int most = 16 * sm_count();
  const int grid = blocks < most ? static_cast<int>(blocks) : most;
  if (dtype == TNX_BF16)
    return launch("combining experts", combine_kernel<__nv_bfloat16>, grid, 256, 0, 1, stream, part, pos,
                  static_cast<__nv_bfloat16*>(out), static_cast<long long>(ld_out), tokens, top_k, cols, splits, slice);
  return launch("combining experts", combine_kernel<__half>, grid, 256, 0, 1, stream, part, pos,
                static_cast<__half*>(out), static_cast<long long>(ld_out), tokens, top_k, cols, splits, slice);
}

RowsParams rows_params(const tnx_moe_problem& p, const Plan& plan, int32_t* status) {
  RowsParams g = {};
  g.plan = plan;
  g.activation = p.activation;
  g.status = status;
  g.timeout_ns = bounded_wait_limit_ns();
  return g;
}
// Cuts K into `splits` slices, none of them empty.
void split_k(RowsParams* g, int k, int splits) {
  const int num_kb = cdiv(k, kTileK);
  g->k = k;
  g->num_kb = num_kb;
  g->kb_per_split = cdiv(num_kb, splits);
  g->splits = cdiv(num_kb, g->kb_per_split);
}

template <typename T>
int run_stream(const tnx_moe_problem& p, const Layout& l, const void* x, const void* w12, const void* w3,
               const void* ids, const float* weights, T* y, char* ws, cudaStream_t stream) {
  StreamParams q = {};
  q.ids = ids;
  q.wide = p.wide_ids;
  q.experts = p.experts;
  q.pairs = l.pairs;
  q.top_k = p.top_k;
  q.weights = weights;
  q.activation = p.activation;
  q.x = x;
  q.ld_x = p.stride_x;
  q.w = w12;
  q.expert_pitch = p.stride_w12e;
  q.row_pitch = p.stride_w12k;
  q.k = p.d_model;
  q.cols = 2 * p.d_ff;
  q.slices = l.up_slices;
  q.slice_k = l.up_slice_k;
  q.out = reinterpret_cast<float*>(ws);
  dim3 grid(static_cast<unsigned>(cdiv(q.cols, kStreamCols) * q.slices), static_cast<unsigned>(l.pairs));
  int rc = launch("streamed gate/up product", stream_kernel<T, false>, grid, dim3(kStreamThreads), 0, 1, stream, q);
  if (rc != TNX_OK) return rc;
  q.parts = q.out;
  q.parts_n = q.slices;
  q.w = w3;
  q.expert_pitch = p.stride_w3e;
  q.row_pitch = p.stride_w3k;
  q.k = p.d_ff;
  q.cols = p.n_out;
  q.slices = l.down_slices;
  q.slice_k = l.down_slice_k;
  q.out = reinterpret_cast<float*>(ws + l.up_bytes);
  grid.x = static_cast<unsigned>(cdiv(q.cols, kStreamCols) * q.slices);
  rc = launch("streamed down product", stream_kernel<T, true>, grid, dim3(kStreamThreads), 0, 1, stream, q);
  if (rc != TNX_OK) return rc;
  return launch("joining streamed products", stream_join_kernel<T>,
                dim3(static_cast<unsigned>(cdiv(p.n_out, 32)), static_cast<unsigned>(p.tokens)), dim3(32, 8), 0, 1, stream,
                q, y, static_cast<long long>(p.stride_y));
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
  out->tile_rows = kTileN;
  out->max_tiles = l.max_tiles;
  const int64_t keep = l.plan_bytes + l.hidden_bytes;
  out->saved_bytes = keep + l.gu_bytes;
  out->workspace_bytes =
      l.stream ? l.up_bytes + l.down_bytes : l.part_bytes + l.chunk_bytes + l.x_bytes + (problem->train ? 0 : keep);
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
  if (l.stream)
    return p.dtype == TNX_BF16
               ? run_stream(p, l, x, w12, w3, ids, weights, static_cast<__nv_bfloat16*>(y), ws, s)
               : run_stream(p, l, x, w12, w3, ids, weights, static_cast<__half*>(y), ws, s);
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
  RowsParams g = rows_params(p, plan, status_word);
  split_k(&g, p.d_model, 1);
  g.cols = 2 * p.d_ff;
  g.out = hidden;
  g.gu = static_cast<float*>(gu);
  CUtensorMap tw;
  RowsMaps rows;
  rc = weights_map(&tw, &g, p, w12, 2 * p.d_ff, p.d_model, p.stride_w12k, p.stride_w12e);
  if (rc == TNX_OK && l.gather) {
    rc = make_tmap_2d(&rows.m[3], x, p.dtype, p.d_model, p.tokens, p.stride_x, 64, 1, true);
    rows.m[0] = rows.m[1] = rows.m[2] = rows.m[3];
  } else if (rc == TNX_OK) {
    rc = rows_maps(&rows, xp, p.dtype, p.d_model, l.max_rows);
  }
  if (rc != TNX_OK) return rc;
  rc = p.train    ? launch_rows<kGateUpKeep>(p, l, tw, rows, g, s)
       : l.gather ? launch_rows<kGateUpGather>(p, l, tw, rows, g, s)
                  : launch_rows<kGateUp>(p, l, tw, rows, g, s);
  if (rc != TNX_OK) return rc;

  // O = H W3
  split_k(&g, p.d_ff, l.down_splits);
  g.cols = p.n_out;
  g.out = part;
  rc = weights_map(&tw, &g, p, w3, p.n_out, p.d_ff, p.stride_w3k, p.stride_w3e);
  if (rc == TNX_OK) rc = rows_maps(&rows, hidden, p.dtype, p.d_ff, l.max_rows);
  if (rc == TNX_OK) rc = launch_rows<kDown>(p, l, tw, rows, g, s);
  if (rc != TNX_OK) return rc;
  return run_combine(p.dtype, part, plan.pos, y, p.stride_y, p.tokens, p.top_k, p.n_out, g.splits, l.max_rows, s);
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
  float* gu = reinterpret_cast<float*>(keep + l.plan_bytes + l.hidden_bytes);
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

  // dH = dY W3^T; dGU and the routing weights' gradient from it
  RowsParams g = rows_params(p, plan, status_word);
  CUtensorMap tw;
  RowsMaps rows;
  if (hidden_grad) {
    split_k(&g, p.n_out, 1);
    g.cols = p.d_ff;
    g.out = dgu;
    g.gu = gu;
    g.dw_part = dw_part;
    g.dw_parts = l.dw_parts;
    rc = make_tmap_3d(&tw, w3, p.dtype, p.n_out, p.d_ff, p.experts, p.stride_w3k, p.stride_w3e, 64, kRows, true);
    if (rc == TNX_OK) rc = rows_maps(&rows, dyp, p.dtype, p.n_out, l.max_rows);
    if (rc == TNX_OK) rc = launch_rows<kDHidden>(p, l, tw, rows, g, s);
    if (rc == TNX_OK && dweights != nullptr)
      rc = launch("routing weights' gradient", weight_grad_kernel, cdiv(l.pairs, 16), 256, 0, 1, s,
                  static_cast<const float*>(dw_part), static_cast<const int*>(plan.pos), dweights, l.pairs, l.dw_parts);
    if (rc != TNX_OK) return rc;
  }
  if (dx != nullptr) {
    split_k(&g, static_cast<int>(two_f), l.dx_splits);
    g.cols = p.d_model;
    g.out = dx_part;
    rc = make_tmap_3d(&tw, w12, p.dtype, two_f, p.d_model, p.experts, p.stride_w12k, p.stride_w12e, 64, kRows, true);
    if (rc == TNX_OK) rc = rows_maps(&rows, dgu, p.dtype, static_cast<int>(two_f), l.max_rows);
    if (rc == TNX_OK) rc = launch_rows<kDX>(p, l, tw, rows, g, s);
    if (rc == TNX_OK)
      rc = run_combine(p.dtype, dx_part, plan.pos, dx, p.d_model, p.tokens, p.top_k, p.d_model, g.splits, l.max_rows, s);
    if (rc != TNX_OK) return rc;
  }
  if (dw12 != nullptr)
    rc = run_wgrad(p, l, plan, xp, p.d_model, dgu, static_cast<int>(two_f), dw12, status_word, s);
  if (rc == TNX_OK && dw3 != nullptr) rc = run_wgrad(p, l, plan, hidden, p.d_ff, dyp, p.n_out, dw3, status_word, s);
  return rc;
}

}  // extern "C"
