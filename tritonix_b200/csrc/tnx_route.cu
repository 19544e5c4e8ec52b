// Routing of tokens to experts, and its gradient.
//     s = softmax(l) or sigmoid(l)                 one score per expert
//     c = s + bias                                 what experts are chosen by
//     groups of consecutive experts: a group's score is the sum of its two best c; only experts of
//     the `top_groups` best groups can be chosen
//     ids = the top_k experts by c, best first, ties to the lowest index
//     w = scale * s[ids] (/ sum of s[ids] when renormalised)
//
// One warp per token: a token's experts are spread over the lanes (expert j*32 + lane in register
// j).  A lane sorts its own experts once (64-bit keys: the choice's order-preserving integer above,
// the expert's number below); a pick then is the largest of the lanes' heads (two redux.sync), and
// the lane that had it moves up its list.  Forward reads each logit once and writes top_k weights
// and ids.  At 32768 tokens x 256 experts in 8 groups this is 36 MB (5.5 us at the measured copy
// rate), but instructions bound the kernel: some 1350 per token (57 us), after 2100 with a search of all
// registers for every pick (105 us).
//
// Which experts are chosen must not depend on how an exponential is rounded.  Without a bias the
// logits themselves order the experts exactly.  With a bias or with groups the fp32 choices carry
// a bound on their error, and a token for which two choices that decide anything are closer
// than that bound (unless they are copies of one another) is chosen again in 64 bits.
#include <cuda_runtime.h>
#include <math_constants.h>

#include "tnx_elem.cuh"
#include "tnx_internal.h"

namespace tnx {

namespace {

constexpr int kWarps = 4;  // tokens of a block
constexpr int kMaxExperts = 512;
constexpr int kMaxTokens = 2147483647 - (kWarps - 1);
constexpr int kMaxPicks = 32;  // lane i keeps pick i
constexpr unsigned kAll = 0xffffffffu;

struct RouteParams {
  int tokens, experts, top_k, groups, top_groups, scoring, renormalize;
  unsigned group_size, group_inv;  // experts of a group; ceil(2^20 / group_size): e / group_size = e * inv >> 20
  float scale;
  long long ld;  // row pitch of the logits in elements
  const void* logits;
  const float* bias;
  float* weights;
  int* ids;
  // backward
  const int* chosen;
  const float* dweights;
  void* dlogits;
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Integers in the order of the floats: NaN below everything, 0 is kept for "cannot be chosen".
__device__ __forceinline__ unsigned order_key(float v) {
  const int u = __float_as_int(v + 0.f);  // (-0 becomes +0)
  const unsigned k = static_cast<unsigned>(u ^ ((u >> 31) | static_cast<int>(0x80000000u)));
  return v != v ? 1u : k;
}
__device__ __forceinline__ float key_value(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  if (v != v) return 1ull;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v + 0.0));
  return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}
__device__ __forceinline__ unsigned warp_key_max(unsigned k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ unsigned long long warp_key_max(unsigned long long k) {
  const unsigned hi = __reduce_max_sync(kAll, static_cast<unsigned>(k >> 32));
  const unsigned lo = __reduce_max_sync(kAll, static_cast<unsigned>(k >> 32) == hi ? static_cast<unsigned>(k) : 0u);
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

// Scores of the lane's experts in F = float or double.  A row of -infinities alone scores 0.
// TO_CHOOSE: a NaN is left out of the softmax's sum, so that the others can still be told apart by
// their scores, and infinity is the limit of a large logit.
template <typename F, int VPT, bool TO_CHOOSE = false>
__device__ __forceinline__ void scores(const float (&l)[VPT], int experts, int lane, bool softmax, float row_max,
                                       F (&s)[VPT]) {
  if (softmax) {
    F sum = 0;
    const float top = row_max == -CUDART_INF_F ? 0.f : row_max;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      s[j] = j * 32 + lane < experts ? exp(static_cast<F>(l[j]) - static_cast<F>(top)) : static_cast<F>(0);
      if (TO_CHOOSE && l[j] == top) s[j] = static_cast<F>(1);  // (infinity minus infinity)
      if (!TO_CHOOSE || s[j] == s[j]) sum += s[j];
    }
    sum = warp_sum(sum);
    const F inv = sum == static_cast<F>(0) ? static_cast<F>(0) : static_cast<F>(1) / sum;
#pragma unroll
    for (int j = 0; j < VPT; ++j) s[j] *= inv;
  } else {
#pragma unroll
    for (int j = 0; j < VPT; ++j) s[j] = static_cast<F>(1) / (static_cast<F>(1) + exp(-static_cast<F>(l[j])));
  }
}

// sigmoid(l) and 1 - sigmoid(l), both to a few units in the last place however far l is from 0.
__device__ __forceinline__ float2 sigmoid_and_rest(float l) {
  const float e = expf(-fabsf(l)), near = 1.f / (1.f + e), far = e * near;
  return l >= 0.f ? make_float2(near, far) : make_float2(far, near);
}
// A renormalised sigmoid's weight of the lane's pick, before the division by the warp's sum of them,
// for picks whose scores themselves have a sum below kFewScores: sigmoid(l) / exp(m), m the largest of
// the picks' min(l, 0), so that it does not matter whether fp32 holds the scores (below l = -103 it
// does not).  Scores that are 0 in 64 bits (1 / (1 + exp(-l)) with an exponential that overflows:
// l < -709.78, a type's lowest value among them) stay 0.  (Above the limit scores that fp32 does not
// hold are weights below 2^-125.)
constexpr float kFewScores = 1e-7f;
__device__ __forceinline__ float sigmoid_share(float l, bool picked) {
  const bool zero = !picked || l < -709.78265f;
  const float a = fminf(l, 0.f);
  const float m = warp_max(zero ? -CUDART_INF_F : a);
  if (zero) return 0.f;
  // (the rounding of a - m would be an error of the weight's 80 units in the last place at a - m = -80)
  const float d = a - m, b = d - a, rest = (a - (d - b)) - (m + b);
  const float e = expf(d);
  return fmaf(e, rest, e) / (1.f + expf(-fabsf(l)));
}

// Scores that only take part in the choice: fast exponential and division (see the bound on their
// error in route_kernel).  False where the row's sum is not a number, and no score with it: a logit is
// NaN or infinity.
template <int VPT>
__device__ __forceinline__ bool quick_scores(const float (&l)[VPT], int experts, int lane, bool softmax, float row_max,
                                             float (&s)[VPT]) {
  if (softmax) {
    float sum = 0.f;
    const float top = row_max == -CUDART_INF_F ? 0.f : row_max;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      s[j] = j * 32 + lane < experts ? __expf(l[j] - top) : 0.f;
      sum += s[j];
    }
    sum = warp_sum(sum);
    const float inv = sum == 0.f ? 0.f : __fdividef(1.f, sum);
#pragma unroll
    for (int j = 0; j < VPT; ++j) s[j] *= inv;
    return sum == sum;
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j) s[j] = __fdividef(1.f, 1.f + __expf(-l[j]));
  return true;
}

// Which groups stay open, as a bit mask the whole warp agrees on, by the sum of each group's two
// best choices (its only one in a group of one).  `c` is the warp's shared copy of the choices.
// Lanes are dealt out to the groups in equal numbers of a power of two.  *gap: how far the worst
// open group is from the best closed one (infinite when no group is closed).
template <typename F>
__device__ __forceinline__ unsigned open_groups(const F* c, int groups, int size, int top_groups, int lane, F* gap) {
  int bits = 0;
  while ((2 << bits) * groups <= 32) ++bits;
  const int share = 1 << bits;
  const int g = lane >> bits;
  const F low = static_cast<F>(-CUDART_INF_F);
  F first = low, second = low;
  if (g < groups)
    for (int i = lane & (share - 1); i < size; i += share) {
      const F v = c[g * size + i];
      if (v > first) {
        second = first;
        first = v;
      } else if (v > second) {
        second = v;
      }
    }
  for (int o = 1; o < share; o <<= 1) {
    const F f2 = __shfl_xor_sync(kAll, first, o), s2 = __shfl_xor_sync(kAll, second, o);
    const F worse = first < f2 ? first : f2;
    first = first < f2 ? f2 : first;
    second = second < s2 ? s2 : second;
    second = second < worse ? worse : second;
  }
  const F total = size > 1 ? first + second : first;
  // lane g holds the key of group g
  const F mine = __shfl_sync(kAll, total, (lane * share) & 31);
  auto key = lane < groups ? order_key(mine) : static_cast<decltype(order_key(mine))>(0);
  unsigned open = 0;
  F last = 0;
  for (int i = 0; i < top_groups; ++i) {
    const auto best = warp_key_max(key);
    const int at = __ffs(__ballot_sync(kAll, key == best)) - 1;
    open |= 1u << at;
    last = __shfl_sync(kAll, mine, at);
    if (lane == at) key = 0;
  }
  *gap = static_cast<F>(CUDART_INF_F);
  const auto next = warp_key_max(key);
  if (next != 0) {
    const int at = __ffs(__ballot_sync(kAll, key == next)) - 1;
    *gap = last - __shfl_sync(kAll, mine, at);
  }
  return open;
}

// The group of expert e < 512 (with one group its number is not asked for: all bits are set).
__device__ __forceinline__ unsigned group_of(const RouteParams& p, int e) {
  return p.groups == 1 ? 0u : static_cast<unsigned>(e) * p.group_inv >> 20;
}

// The same choice in 64 bits, for tokens that fp32 cannot tell apart.  Returns pick `lane`'s expert.
// `logits` and `shared` are the warp's, and do not overlap.
template <int VPT>
__device__ __noinline__ int choose_exactly(const float* logits, const RouteParams& p, int lane, float row_max,
                                           double* shared) {
  float l[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) l[j] = logits[j * 32 + lane];
  double c[VPT];
  scores<double, VPT, true>(l, p.experts, lane, p.scoring == TNX_SCORE_SOFTMAX, row_max, c);
  unsigned open = kAll;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int e = j * 32 + lane;
    if (e < p.experts && p.bias != nullptr) c[j] += static_cast<double>(p.bias[e]);
  }
  if (p.groups > 1) {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (j * 32 + lane < p.experts) shared[j * 32 + lane] = c[j];
    __syncwarp();
    double gap;
    open = open_groups(shared, p.groups, static_cast<int>(p.group_size), p.top_groups, lane, &gap);
    __syncwarp();
  }
  unsigned long long key[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int e = j * 32 + lane;
    key[j] = e < p.experts && ((open >> group_of(p, e)) & 1u) ? order_key(c[j]) : 0ull;
  }
  int mine = 0;
  for (int i = 0; i < p.top_k; ++i) {
    unsigned long long best = 0;
    int at = kMaxExperts;
#pragma unroll
    for (int j = VPT - 1; j >= 0; --j)
      if (key[j] >= best) {
        best = key[j];
        at = j * 32 + lane;
      }
    const unsigned long long top = warp_key_max(best);
    const int e = __reduce_min_sync(kAll, best == top ? static_cast<unsigned>(at) : static_cast<unsigned>(kMaxExperts));
    if (lane == i) mine = e;
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (e == j * 32 + lane) key[j] = 0;
  }
  return mine;
}

// Sorts a lane's keys, largest first (Batcher's odd-even merge sort).  Every loop has a constant
// trip count and every comparison of indices folds, so that the keys stay in registers.
template <int N>
__device__ __forceinline__ void sort_keys(unsigned long long (&k)[N]) {
#pragma unroll
  for (int lp = 0; (1 << lp) < N; ++lp) {
#pragma unroll
    for (int lq = lp; lq >= 0; --lq) {
      const int p = 1 << lp, q = 1 << lq;
#pragma unroll
      for (int t = 0; t + q < N; ++t) {
        const int from = q % p;  // merges start here: the first element of a run, or past its first q
        if (t >= from && (t - from) % (2 * q) < q && t / (2 * p) == (t + q) / (2 * p)) {
          const unsigned long long a = k[t], b = k[t + q];
          k[t] = a > b ? a : b;
          k[t + q] = a > b ? b : a;
        }
      }
    }
  }
}

template <typename T, int VPT>
__global__ void __launch_bounds__(kWarps * 32, VPT <= 8 ? 8 : 4) route_kernel(const __grid_constant__ RouteParams p) {
  // Per warp: the logits by expert, and the choices (as doubles for a token that needs them exact).
  __shared__ float logits[kWarps][VPT * 32];
  __shared__ double shared[kWarps][VPT * 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int token = blockIdx.x * kWarps + warp;
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.ld;
  float* sh_logit = logits[warp];
  float* sh_choice = reinterpret_cast<float*>(shared[warp]);
  // (no branches in the unrolled loops: experts that do not exist are read at the last one)
  float l[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) l[j] = elem::to_float(row[min(j * 32 + lane, p.experts - 1)]);
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    if (j * 32 + lane >= p.experts) l[j] = -CUDART_INF_F;
    sh_logit[j * 32 + lane] = l[j];
  }
  const bool softmax = p.scoring == TNX_SCORE_SOFTMAX, biased = p.bias != nullptr;
  float row_max = -CUDART_INF_F;
  if (softmax) {
#pragma unroll
    for (int j = 0; j < VPT; ++j) row_max = fmaxf(row_max, l[j]);
    row_max = warp_max(row_max);
  }
  float eps = 0.f;
  unsigned open = kAll;
  bool unsure = false;
  if (biased || p.groups > 1) {  // (otherwise the logits order the experts)
    float c[VPT];
    unsure = !quick_scores<VPT>(l, p.experts, lane, softmax, row_max, c);
    float top_score = 1.f;
    if (softmax) {
      top_score = c[0];
#pragma unroll
      for (int j = 1; j < VPT; ++j) top_score = fmaxf(top_score, c[j]);
      top_score = warp_max(top_score);
    }
    float far = 0.f;  // largest |bias|
    if (biased) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const float b = p.bias[min(j * 32 + lane, p.experts - 1)];
        c[j] += b;
        far = fmaxf(far, fabsf(b));
      }
      far = warp_max(far);
    }
    // The largest error a choice can have.  Relative to the score: the exponential, the division and
    // the sum are good to a few units in the last place each, 2^-19 together.  Rounding x = l - max
    // (or -l) and its product with log2(e) puts an error of 2 |x| 2^-24 into the exponent; score times
    // |x| is at most 0.37 (softmax, where the score is at most exp(x)) or 0.28 (sigmoid, whose
    // derivative is s (1 - s)): 1.2e-7 is more than twice that.  The bias's addition rounds once more.
    eps = 1.91e-6f * top_score + 1.2e-7f + 6e-8f * (top_score + far);
    if (p.groups > 1) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) sh_choice[j * 32 + lane] = c[j];
      __syncwarp();
      float gap;
      open = open_groups(sh_choice, p.groups, static_cast<int>(p.group_size), p.top_groups, lane, &gap);
      unsure = unsure || !(gap > 4.f * eps);  // (two choices on each side)
    }
    if (biased) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) l[j] = c[j];
    }
  }
  __syncwarp();
  unsigned long long key[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int e = j * 32 + lane;
    key[j] = (static_cast<unsigned long long>(order_key(l[j])) << 32) | (0xffffffffu - static_cast<unsigned>(e));
    if (e >= p.experts) key[j] = 0ull;
  }
  if (p.groups > 1) {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (!((open >> group_of(p, j * 32 + lane)) & 1u)) key[j] = 0ull;
  }
  sort_keys<VPT>(key);

  int mine = 0;  // pick `lane`
  float last = 0.f;
  int last_e = 0;
  const int rounds = p.top_k + (biased ? 1 : 0);  // one more to see the best that is left out
  for (int i = 0; i < rounds && !unsure; ++i) {
    const unsigned long long top = warp_key_max(key[0]);
    if (top == 0) break;  // (only past the last pick: nothing is left out)
    const int e = static_cast<int>(0xffffffffu - static_cast<unsigned>(top));
    if (key[0] == top) {
#pragma unroll
      for (int j = 0; j + 1 < VPT; ++j) key[j] = key[j + 1];
      key[VPT - 1] = 0ull;
    }
    if (biased) {
      const float v = key_value(static_cast<unsigned>(top >> 32));
      // (copies of one another are in order already)
      if (i > 0 && !(last - v > 2.f * eps))
        unsure = !(sh_logit[e] == sh_logit[last_e] && p.bias[e] == p.bias[last_e]);
      last = v;
      last_e = e;
    }
    if (lane == i) mine = e;
  }
  float my_logit, my_score;
  if (unsure) mine = choose_exactly<VPT>(sh_logit, p, lane, row_max, shared[warp]);
  my_logit = sh_logit[mine];
  if (softmax) {
    my_score = 0.f;
    if (!p.renormalize) {  // (the quick scores will not do: a sum of accurate exponentials)
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (j * 32 + lane < p.experts) sum += expf(sh_logit[j * 32 + lane] - row_max);
      sum = warp_sum(sum);
      my_score = row_max == -CUDART_INF_F ? 0.f : expf(my_logit - row_max) / sum;
    }
  } else {
    my_score = sigmoid_and_rest(my_logit).x;
  }

  const bool picked = lane < p.top_k;
  float w = my_score;
  if (p.renormalize) {
    if (softmax) {
      // a softmax over the picks alone: the same ratio, and no score underflows in it
      const float top = warp_max(picked ? my_logit : -CUDART_INF_F);
      w = picked ? expf(my_logit - (top == -CUDART_INF_F ? 0.f : top)) : 0.f;
    }
    float sum = warp_sum(picked ? w : 0.f);
    if (!softmax && sum < kFewScores) {
      w = sigmoid_share(my_logit, picked);
      sum = warp_sum(w);
    }
    w = sum == 0.f ? 0.f : w / sum;
  }
  if (picked) {
    const long long at = static_cast<long long>(token) * p.top_k + lane;
    p.weights[at] = w * p.scale;
    p.ids[at] = mine;
  }
}

// Gradient of the logits from that of the weights (a warp per token).  With s the scores and
// r = w / scale:
//   softmax, renormalised   dl_i = scale r_i (dw_i - sum_j dw_j r_j)      for picks, 0 elsewhere
//   sigmoid, renormalised   the same times (1 - s_i)
//   sigmoid                 dl_i = scale dw_i s_i (1 - s_i)
//   softmax                 dl_e = scale p_e ([e picked] dw_e - sum_j dw_j p_j)   for every expert
// The sums run over the picks.  Only the last form reads the whole row again.
template <typename T, int VPT>
__global__ void __launch_bounds__(kWarps * 32) route_backward_kernel(const RouteParams p) {
  const int lane = threadIdx.x & 31;
  const int token = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (token >= p.tokens) return;
  const T* row = static_cast<const T*>(p.logits) + token * p.ld;
  const bool softmax = p.scoring == TNX_SCORE_SOFTMAX;
  const long long at = static_cast<long long>(token) * p.top_k + lane;
  int e = lane < p.top_k ? p.chosen[at] : -1;
  if (e >= p.experts) e = -1;
  const bool picked = e >= 0;
  const float dw = picked ? p.dweights[at] * p.scale : 0.f;
  const float logit = picked ? elem::to_float(row[e]) : -CUDART_INF_F;

  float out[VPT], base = 0.f, g = 0.f;  // g: this lane's pick's gradient, less `base` times the row's scores
#pragma unroll
  for (int j = 0; j < VPT; ++j) out[j] = 0.f;
  if (softmax && !p.renormalize) {
    float l[VPT], top = -CUDART_INF_F;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      l[j] = j * 32 + lane < p.experts ? elem::to_float(row[j * 32 + lane]) : -CUDART_INF_F;
      top = fmaxf(top, l[j]);
    }
    top = warp_max(top);
    scores<float, VPT>(l, p.experts, lane, true, top, out);
    float mine = 0.f;  // score of this lane's pick
    for (int i = 0; i < p.top_k; ++i) {
      const int pick = __shfl_sync(kAll, e, i);
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (pick == j * 32 + lane) v = out[j];
      v = __shfl_sync(kAll, v, pick & 31);
      if (lane == i) mine = v;
    }
    base = warp_sum(picked ? dw * mine : 0.f);
    g = dw;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const float score = out[j];
      float d = 0.f;
      for (int i = 0; i < p.top_k; ++i) {
        const int pick = __shfl_sync(kAll, e, i);
        const float dv = __shfl_sync(kAll, g, i);
        if (pick == j * 32 + lane) d = dv;
      }
      out[j] = score * (d - base);
    }
  } else {
    float r, sum, rest = 1.f;  // rest: 1 - s
    if (softmax) {
      const float top = warp_max(logit);
      r = picked ? expf(logit - (top == -CUDART_INF_F ? 0.f : top)) : 0.f;
      sum = warp_sum(r);
    } else {
      const float2 s = sigmoid_and_rest(logit);
      r = picked ? s.x : 0.f;
      rest = s.y;
      sum = 1.f;
      if (p.renormalize) {
        sum = warp_sum(r);
        if (sum < kFewScores) {
          r = sigmoid_share(logit, picked);
          sum = warp_sum(r);
        }
      }
    }
    if (p.renormalize) {
      r = sum == 0.f ? 0.f : r / sum;
      base = warp_sum(picked ? dw * r : 0.f);
    }
    g = r * (dw - base) * rest;
    for (int i = 0; i < p.top_k; ++i) {
      const int pick = __shfl_sync(kAll, e, i);
      const float v = __shfl_sync(kAll, g, i);
#pragma unroll
      for (int j = 0; j < VPT; ++j)
        if (pick == j * 32 + lane) out[j] = v;
    }
  }
  T* drow = static_cast<T*>(p.dlogits) + static_cast<long long>(token) * p.experts;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
    if (j * 32 + lane < p.experts) drow[j * 32 + lane] = elem::from_float<T>(out[j]);
}

using RouteFn = void (*)(const RouteParams);

template <typename T>
RouteFn pick_experts(int experts, bool backward) {
  if (experts <= 32) return backward ? route_backward_kernel<T, 1> : route_kernel<T, 1>;
  if (experts <= 64) return backward ? route_backward_kernel<T, 2> : route_kernel<T, 2>;
  if (experts <= 128) return backward ? route_backward_kernel<T, 4> : route_kernel<T, 4>;
  if (experts <= 256) return backward ? route_backward_kernel<T, 8> : route_kernel<T, 8>;
  return backward ? route_backward_kernel<T, 16> : route_kernel<T, 16>;
}
RouteFn pick_route(int dtype, int experts, bool backward) {
  if (dtype == TNX_F32) return pick_experts<float>(experts, backward);
  if (dtype == TNX_F16) return pick_experts<__half>(experts, backward);
  return pick_experts<__nv_bfloat16>(experts, backward);
}

int route_check(const tnx_route_problem* p) {
  if (p == nullptr) {
    set_error("problem is NULL");
    return TNX_ERR_INVALID;
  }
  if (p->dtype < TNX_F16 || p->dtype > TNX_F32) {
    set_error("unknown dtype %d", p->dtype);
    return TNX_ERR_INVALID;
  }
  // (the number of a block's last token is an int too)
  if (p->tokens < 0 || p->tokens > kMaxTokens || p->experts < 1 || p->experts > kMaxExperts) {
    set_error("routing needs 0 to %d tokens and 1 <= experts <= %d (got %d tokens, %d experts)", kMaxTokens, kMaxExperts,
              p->tokens, p->experts);
    return TNX_ERR_INVALID;
  }
  if (p->groups < 1 || p->groups > 32 || p->experts % p->groups != 0 || p->top_groups < 1 ||
      p->top_groups > p->groups) {
    set_error("groups must divide the experts, be at most 32, and hold 1 <= top_groups <= groups (got %d experts, "
              "%d groups, %d of them open)", p->experts, p->groups, p->top_groups);
    return TNX_ERR_INVALID;
  }
  const int open = p->experts / p->groups * p->top_groups;
  if (p->top_k < 1 || p->top_k > kMaxPicks || p->top_k > open) {
    set_error("top_k must be in [1, %d] and at most the %d experts that can be chosen, got %d", kMaxPicks, open,
              p->top_k);
    return TNX_ERR_INVALID;
  }
  if (p->scoring != TNX_SCORE_SOFTMAX && p->scoring != TNX_SCORE_SIGMOID) {
    set_error("unknown scoring %d", p->scoring);
    return TNX_ERR_INVALID;
  }
  if (p->stride_logits < 0) {
    set_error("negative strides are not supported");
    return TNX_ERR_INVALID;
  }
  return TNX_OK;
}

RouteParams route_params(const tnx_route_problem& q) {
  RouteParams p = {};
  p.tokens = q.tokens;
  p.experts = q.experts;
  p.top_k = q.top_k;
  // (all groups open: the groups decide nothing)
  p.groups = q.top_groups == q.groups ? 1 : q.groups;
  p.top_groups = q.top_groups == q.groups ? 1 : q.top_groups;
  p.group_size = static_cast<unsigned>(q.experts / p.groups);
  p.group_inv = ((1u << 20) + p.group_size - 1) / p.group_size;
  p.scoring = q.scoring;
  p.renormalize = q.renormalize;
  p.scale = q.scale;
  p.ld = q.stride_logits;
  return p;
}

int route_launch(RouteFn fn, const RouteParams& p, void* stream) {
  fn<<<(p.tokens + kWarps - 1) / kWarps, kWarps * 32, 0, static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return TNX_OK;
  set_error("routing: launch failed: %s", cudaGetErrorString(e));
  return TNX_ERR_CUDA;
}

}  // namespace
}  // namespace tnx

extern "C" {

int tnx_route_experts(const tnx_route_problem* problem, const void* logits, const float* bias, float* weights,
                      int32_t* ids, void* stream) {
  using namespace tnx;
  const int rc = route_check(problem);
  if (rc != TNX_OK) return rc;
  if (problem->tokens == 0) return TNX_OK;
  if (logits == nullptr || weights == nullptr || ids == nullptr) {
    set_error("NULL operand pointer");
    return TNX_ERR_INVALID;
  }
  RouteParams p = route_params(*problem);
  p.logits = logits;
  p.bias = bias;
  p.weights = weights;
  p.ids = ids;
  return route_launch(pick_route(problem->dtype, problem->experts, false), p, stream);
}

int tnx_route_experts_backward(const tnx_route_problem* problem, const void* logits, const int32_t* ids,
                               const float* dweights, void* dlogits, void* stream) {
  using namespace tnx;
  const int rc = route_check(problem);
  if (rc != TNX_OK) return rc;
  if (problem->tokens == 0) return TNX_OK;
  if (logits == nullptr || ids == nullptr || dweights == nullptr || dlogits == nullptr) {
    set_error("NULL operand pointer");
    return TNX_ERR_INVALID;
  }
  RouteParams p = route_params(*problem);
  p.logits = logits;
  p.chosen = ids;
  p.dweights = dweights;
  p.dlogits = dlogits;
  return route_launch(pick_route(problem->dtype, problem->experts, true), p, stream);
}

}  // extern "C"
