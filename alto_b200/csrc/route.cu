// Routing of tokens to experts, its gradient, and the row plan of the padded token buffer.
//
//   score   softmax or sigmoid of the token's logits
//   choice  the top_k largest keys, key = score + bias (the logit itself where that is the same order: no bias and groups
//           judged by one expert); with groups, only experts of the groups_kept best groups, a group's score the sum of
//           its one or two largest keys; the lowest index first among equals
//   weights scale * score of the chosen, over the sum of the chosen scores when renormalised
//
// The choice is made as if keys had 64 bits.  Keys are computed in fp32; where two that a decision separates are nearer
// than fp32 can tell (and not equal because their inputs are), the token is done again in double.
#include "common.cuh"

namespace altob200 {

struct RouteArgs {
  const void* logits;
  const float* bias;     // or NULL
  int32_t* ids;          // [tokens, k]
  float* weights;        // [tokens, k]
  int64_t tokens, ld;
  int32_t experts, k, sigmoid, groups, kept, group_top, renorm;
  float scale;
};

static constexpr int ROUTE_MAX_K = 16, ROUTE_MAX_E = 512, ROUTE_MAX_GROUPS = 32;
static constexpr unsigned FULL = 0xFFFFFFFFu;

template <bool BF16>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
  if constexpr (BF16) return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p) + i));
  else return __ldg(reinterpret_cast<const float*>(p) + i);
}

// Unsigned words in the order of the floats; a NaN above everything, 0 below everything.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = f2u(v);
  if (v != v) return 0xFFFFFFFFu;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  if (v != v) return ~0ull;
  return (b >> 63) ? ~b : (b | (1ull << 63));
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}
template <class F>
__device__ __forceinline__ F warp_add(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ uint32_t warp_max_key(uint32_t v) { return __reduce_max_sync(FULL, v); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(FULL, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(FULL, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((uint64_t)hi << 32) | lo;
}
template <class F>
struct KeyWord;
template <>
struct KeyWord<float> { using U = uint32_t; };
template <>
struct KeyWord<double> { using U = uint64_t; };

template <class F>
__device__ __forceinline__ F exp_of(F v);
template <>
__device__ __forceinline__ float exp_of<float>(float v) { return expf(v); }
template <>
__device__ __forceinline__ double exp_of<double>(double v) { return exp(v); }

// One token by one warp, lane l holding experts l, l + 32, ...  Lane i < k returns the i-th choice in *chosen.  `keys`
// is the warp's own shared memory (padded: see at()).  Returns whether every decision is certain; F = double always is.
template <class F, bool BF16, int V>
__device__ bool choose(const RouteArgs& a, int64_t row, const float* l, const float* b, bool computed, F* keys, int* chosen) {
  using U = typename KeyWord<F>::U;
  constexpr bool FP32 = sizeof(F) == 4;
  const int lane = threadIdx.x & 31, E = a.experts;
  F key[V];
  bool sure = true;
  if (computed) {
    F m = 0, z = 1;
    if (!a.sigmoid) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (lane + 32 * j < E) top = fmaxf(top, l[j]);
      m = (F)warp_max(top);
      z = 0;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (lane + 32 * j < E) z += exp_of<F>((F)l[j] - m);
      z = warp_add(z);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const F s = a.sigmoid ? (F)1 / ((F)1 + exp_of<F>(-(F)l[j])) : exp_of<F>((F)l[j] - m) / z;
      key[j] = a.bias != nullptr ? s + (F)b[j] : s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = (F)l[j];
  }
  uint32_t allowed = FULL;   // bit g: group g
  int size = E;
  if (a.groups > 1) {
    size = E / a.groups;
    const auto at = [&](int e) { return e + e / size; };   // a word between groups: their lanes read different banks
    __syncwarp();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = lane + 32 * j;
      if (e < E) keys[at(e)] = key[j];
    }
    __syncwarp();
    F best = -INFINITY, second = -INFINITY;
    bool nan = false;
    if (lane < a.groups) {
      for (int i = 0; i < size; ++i) {
        const F v = keys[lane * (size + 1) + i];
        nan = nan || v != v;
        if (v > best) {
          second = best;
          best = v;
        } else if (v > second) {
          second = v;
        }
      }
    }
    F of_group = a.group_top == 2 && size > 1 ? best + second : best;
    if (nan) of_group = NAN;
    const U word = lane < a.groups ? ordered(of_group) : (U)0;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const U other = __shfl_sync(FULL, word, g);
      rank += other > word || (other == word && g < lane) ? 1 : 0;
    }
    allowed = __ballot_sync(FULL, lane < a.groups && rank < a.kept);
    if (FP32 && computed && a.kept < a.groups) {
      // the last group that is kept against the first that is not
      const unsigned last = __ballot_sync(FULL, lane < a.groups && rank == a.kept - 1);
      const unsigned first = __ballot_sync(FULL, lane < a.groups && rank == a.kept);
      const F u = __shfl_sync(FULL, of_group, __ffs(last) - 1), v = __shfl_sync(FULL, of_group, __ffs(first) - 1);
      if (u - v <= (F)1.6e-5f + (F)5e-7f * (F)fabsf((float)u)) sure = false;
    }
  }
  U word[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = lane + 32 * j;
    word[j] = e < E && ((allowed >> (a.groups > 1 ? (e / size) & 31 : 0)) & 1u) ? ordered(key[j]) : (U)0;
  }
  // the next one after the last is looked at too, where there is one
  const int left = (a.groups > 1 ? a.kept * size : E), picks = left > a.k ? a.k + 1 : a.k;
  int mine = 0;
  U mine_word = 0;
  for (int i = 0; i < picks; ++i) {
    U top = word[0];
    int where = lane;
#pragma unroll
    for (int j = 1; j < V; ++j)
      if (word[j] > top) {
        top = word[j];
        where = lane + 32 * j;
      }
    const U best = warp_max_key(top);
    const int e = (int)__reduce_min_sync(FULL, top == best ? (uint32_t)where : 0x7FFFFFFFu);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (lane + 32 * j == e) word[j] = (U)0;
    if (lane == i) {
      mine = e;
      mine_word = best;
    }
  }
  *chosen = mine;
  if constexpr (FP32) {
    if (computed) {
      // neighbours in the order whose keys fp32 cannot tell apart, unless their inputs are the same.  A score is off by
      // at most 7e-6 of itself (the rounding of l - m before the exponential, up to 88 * 2^-24, is the most of it), the
      // sum with the bias by half a step.
      const bool on = lane < picks;
      const float my_l = on ? logit_at<BF16>(a.logits, row + mine) : 0.0f, my_b = on && a.bias != nullptr ? __ldg(a.bias + mine) : 0.0f;
      const float my_key = u2f(mine_word >> 31 ? mine_word & 0x7FFFFFFFu : ~mine_word);
      const float next_l = __shfl_down_sync(FULL, my_l, 1), next_b = __shfl_down_sync(FULL, my_b, 1);
      const float next_key = __shfl_down_sync(FULL, my_key, 1);
      const float room = 1.6e-5f * fmaxf(my_key - my_b, next_key - next_b) + 5e-7f * fabsf(my_key);
      const bool close = lane + 1 < picks && my_key - next_key <= room && !(my_l == next_l && my_b == next_b);
      if (__any_sync(FULL, close)) sure = false;
    }
  }
  return sure;
}

// Weights of the chosen, on lanes i < k (l: the chosen logit).  `m`, `z`: maximum and sum of exponentials
// over all experts, used by the softmax that is not renormalised.  Ratios are formed from the chosen alone, so that they
// hold however small the scores are; a token whose chosen scores are all zero gets zero weights.
__device__ __forceinline__ float chosen_weight(bool on, float l, int sigmoid, int renorm, float m, float z, float* total) {
  *total = 1.0f;
  if (sigmoid) {
    // e^(l - c) / (1 + e^l) with c = min(0, the largest chosen logit): in range for any logits
    const float top = warp_max(on ? l : -INFINITY);
    const float c = renorm && top < 0.0f ? (top == -INFINITY ? 0.0f : top) : 0.0f;
    const float s = !on ? 0.0f : l > 0.0f ? 1.0f / (1.0f + expf(-l)) : expf(l - c) / (1.0f + expf(l));
    if (!renorm) return s;
    *total = warp_add(s);
    return *total == 0.0f ? 0.0f : s / *total;
  }
  if (!renorm) return on && m != -INFINITY ? expf(l - m) / z : 0.0f;
  const float top = warp_max(on ? l : -INFINITY);
  if (top == -INFINITY && !__any_sync(FULL, on && l != l)) return 0.0f;
  const float s = on ? expf(l - top) : 0.0f;
  *total = warp_add(s);
  return s / *total;
}

template <bool BF16, int V>
__global__ void __launch_bounds__(256) route_forward_kernel(RouteArgs a) {
  extern __shared__ double route_smem[];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  double* const scratch = route_smem + (threadIdx.x >> 5) * (a.experts + a.groups);
  const bool computed = a.bias != nullptr || a.group_top > 1;
  float b[V] = {};
  if (a.bias != nullptr)
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (lane + 32 * j < a.experts) b[j] = __ldg(a.bias + lane + 32 * j);
  for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < a.tokens; t += (int64_t)gridDim.x * 8) {
    float l[V];
#pragma unroll
    for (int j = 0; j < V; ++j) l[j] = lane + 32 * j < a.experts ? logit_at<BF16>(a.logits, t * a.ld + lane + 32 * j) : -INFINITY;
    int chosen;
    if (!choose<float, BF16, V>(a, t * a.ld, l, b, computed, reinterpret_cast<float*>(scratch), &chosen))
      choose<double, BF16, V>(a, t * a.ld, l, b, computed, scratch, &chosen);
    const bool on = lane < a.k;
    const float mine = on ? logit_at<BF16>(a.logits, t * a.ld + chosen) : 0.0f;
    float m = 0.0f, z = 1.0f, total;
    if (!a.sigmoid && !a.renorm) {
      m = l[0];
#pragma unroll
      for (int j = 1; j < V; ++j) m = fmaxf(m, l[j]);
      m = warp_max(m);
      z = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (lane + 32 * j < a.experts) z += expf(l[j] - m);
      z = warp_add(z);
    }
    float w = chosen_weight(on, mine, a.sigmoid, a.renorm, m, z, &total);
    if (a.bias != nullptr && !a.sigmoid) {   // a NaN that is not among the chosen makes every score one all the same
      bool nan = false;
#pragma unroll
      for (int j = 0; j < V; ++j) nan = nan || l[j] != l[j];
      if (__any_sync(FULL, nan)) w = NAN;
    }
    if (on) {
      a.ids[t * a.k + lane] = chosen;
      a.weights[t * a.k + lane] = w * a.scale;
    }
  }
}

struct RouteGradArgs {
  const void* logits;
  const int32_t* ids;
  const float* grad;     // [tokens, k]
  void* grad_logits;     // [tokens, experts], the logits' type
  int64_t tokens, ld;
  int32_t experts, k, sigmoid, renorm;
  float scale;
};

//   softmax              dl_e = scale p_e (g_e [chosen] - sum g p)       with p over all experts, or over the chosen when
//                                                                        renormalised (then zero for the others)
//   sigmoid              dl_i = scale s_i (1 - s_i) g_i
//   sigmoid, renormalised dl_i = scale q_i (1 - s_i) (g_i - sum g q)     q = s / sum s
template <bool BF16, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteGradArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < a.tokens; t += (int64_t)gridDim.x * 8) {
    const int64_t row = t * a.ld;
    int id = lane < a.k ? __ldg(a.ids + t * a.k + lane) : -1;
    if (id >= a.experts) id = -1;
    const bool on = id >= 0;
    const float l = on ? logit_at<BF16>(a.logits, row + id) : 0.0f, g = on ? __ldg(a.grad + t * a.k + lane) : 0.0f;
    float m = 0.0f, z = 1.0f, total, all[V] = {};
    const bool dense = !a.sigmoid && !a.renorm;
    if (dense) {
      m = -INFINITY;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        all[j] = lane + 32 * j < a.experts ? logit_at<BF16>(a.logits, row + lane + 32 * j) : -INFINITY;
        m = fmaxf(m, all[j]);
      }
      m = warp_max(m);
      z = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (lane + 32 * j < a.experts) z += expf(all[j] - m);
      z = warp_add(z);
    }
    const float w = chosen_weight(on, l, a.sigmoid, a.renorm, m, z, &total);
    float sum = 0.0f, d;
    if (a.sigmoid) {
      const float rest = 1.0f / (1.0f + expf(l));   // 1 - s
      if (a.renorm) sum = warp_add(on ? g * w : 0.0f);
      d = a.scale * w * rest * (g - sum);
    } else {
      sum = warp_add(on ? g * w : 0.0f);
      d = a.scale * w * (g - sum);
    }
    float out[V];
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = dense && m != -INFINITY ? -a.scale * sum * (expf(all[j] - m) / z) : 0.0f;
    for (int i = 0; i < a.k; ++i) {
      const int e = __shfl_sync(FULL, id, i);
      const float v = __shfl_sync(FULL, d, i);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (lane + 32 * j == e) out[j] = v;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = lane + 32 * j;
      if (e < a.experts) {
        if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(a.grad_logits)[t * a.experts + e] = __float2bfloat16_rn(out[j]);
        else reinterpret_cast<float*>(a.grad_logits)[t * a.experts + e] = out[j];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// row plan: a counting sort of the routed slots by expert, stable, every expert's run padded to `align` rows
// ---------------------------------------------------------------------------------------
struct PlanArgs {
  const void* ids;       // [slots] int32 or int64
  int32_t* token;        // [rows] token of a row, -1: padding
  int32_t* position;     // [rows] routed slot of a row, -1: padding
  int32_t* slot;         // [slots] row of a routed slot, -1: no row
  int32_t* offs;         // [experts] ends of the padded runs
  int32_t* counts;       // [experts] rows without padding
  int32_t* hist;         // [parts][experts] (parts > 1)
  int64_t slots, rows;
  int32_t k, experts, align, wide, parts, per_part;   // per_part: slots of a part, a multiple of 256
};
static constexpr int PLAN_MAX_E = 1024;

__device__ __forceinline__ int plan_id(const PlanArgs& a, int64_t i) {
  if (a.wide) {
    const int64_t v = __ldg(reinterpret_cast<const long long*>(a.ids) + i);
    return v >= 0 && v < a.experts ? (int)v : -1;
  }
  const int v = __ldg(reinterpret_cast<const int32_t*>(a.ids) + i);
  return v >= 0 && v < a.experts ? v : -1;
}

__global__ void __launch_bounds__(256) plan_count_kernel(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  grid_dependency_wait();
  for (int e = threadIdx.x; e < a.experts; e += 256) plan_smem[e] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * a.per_part;
  const int64_t last = first + a.per_part < a.slots ? first + a.per_part : a.slots;
  for (int64_t i = first + threadIdx.x; i < last; i += 256) {
    const int e = plan_id(a, i);
    if (e >= 0) atomicAdd(&plan_smem[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += 256) a.hist[(int64_t)blockIdx.x * a.experts + e] = plan_smem[e];
}

// Part of the slots by one CTA, its eight warps in sequence over per_part / 8 slots each.
__global__ void __launch_bounds__(256) plan_place_kernel(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* const of_warp = plan_smem;                       // [8][experts] counts of the warps, then next rows
  int32_t* const count = plan_smem + 8 * a.experts;         // [experts] rows of an expert
  int32_t* const start = count + a.experts;                 // [experts] its first row
  int32_t* const before = start + a.experts;                // [experts] rows from earlier parts
  __shared__ int32_t scan[256];
  grid_dependency_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, E = a.experts;
  for (int i = tid; i < 8 * E; i += 256) of_warp[i] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * a.per_part + (int64_t)warp * (a.per_part / 8);
  const int64_t stop = first + a.per_part / 8 < a.slots ? first + a.per_part / 8 : a.slots;
  for (int64_t i = first + lane; i < stop; i += 32) {
    const int e = plan_id(a, i);
    if (e >= 0) atomicAdd(&of_warp[warp * E + e], 1);
  }
  __syncthreads();
  // totals and earlier parts, by expert
  for (int e = tid; e < E; e += 256) {
    int all = 0, earlier = 0;
    if (a.parts > 1) {
      for (int p = 0; p < a.parts; ++p) {
        const int c = a.hist[(int64_t)p * E + e];
        if (p == (int)blockIdx.x) earlier = all;
        all += c;
      }
    } else {
      for (int w = 0; w < 8; ++w) all += of_warp[w * E + e];
    }
    count[e] = all;
    before[e] = earlier;
  }
  __syncthreads();
  // first rows: an exclusive sum of the padded counts, E / 256 (rounded up) neighbouring experts a thread
  const int per = (E + 255) / 256;
  int mine = 0;
  for (int j = 0; j < per; ++j) {
    const int e = tid * per + j;
    if (e < E) mine += (count[e] + a.align - 1) / a.align * a.align + (count[e] == 0 ? a.align : 0);
  }
  scan[tid] = mine;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const int v = tid >= o ? scan[tid - o] : 0;
    __syncthreads();
    scan[tid] += v;
    __syncthreads();
  }
  int at = scan[tid] - mine;
  for (int j = 0; j < per; ++j) {
    const int e = tid * per + j;
    if (e < E) {
      start[e] = at;
      at += (count[e] + a.align - 1) / a.align * a.align + (count[e] == 0 ? a.align : 0);
      if (blockIdx.x == 0) {
        a.offs[e] = at;
        a.counts[e] = count[e];
      }
    }
  }
  __syncthreads();
  // next row of every (warp, expert)
  for (int e = tid; e < E; e += 256) {
    int row = start[e] + before[e];
    for (int w = 0; w < 8; ++w) {
      const int c = of_warp[w * E + e];
      of_warp[w * E + e] = row;
      row += c;
    }
  }
  __syncthreads();
  for (int64_t base = first; base < stop; base += 32) {
    const int64_t i = base + lane;
    const int e = i < stop ? plan_id(a, i) : -1;
    const unsigned same = __match_any_sync(FULL, e);
    int row = -1;
    if (e >= 0) row = of_warp[warp * E + e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) of_warp[warp * E + e] += __popc(same);
    __syncwarp();
    if (i < stop) {
      const bool fits = row >= 0 && row < a.rows;
      a.slot[i] = fits ? row : -1;
      if (fits) {
        a.position[row] = (int32_t)i;
        a.token[row] = (int32_t)(i / a.k);
      }
    }
  }
  // padding: the ends of the runs, and what lies behind the last
  for (int e = blockIdx.x; e < E; e += a.parts) {
    const int64_t end = e + 1 < E ? start[e + 1] : (int64_t)start[e] + (count[e] + a.align - 1) / a.align * a.align + (count[e] == 0 ? a.align : 0);
    for (int64_t r = (int64_t)start[e] + count[e] + tid; r < end && r < a.rows; r += 256) {
      a.position[r] = -1;
      a.token[r] = -1;
    }
  }
  const int64_t used = (int64_t)start[E - 1] + (count[E - 1] + a.align - 1) / a.align * a.align + (count[E - 1] == 0 ? a.align : 0);
  for (int64_t r = used + (int64_t)blockIdx.x * 256 + tid; r < a.rows; r += (int64_t)a.parts * 256) {
    a.position[r] = -1;
    a.token[r] = -1;
  }
}

static void plan_split(int64_t slots, int* parts, int* per_part) {
  // one CTA up to 2048 slots, else as many parts as there are SMs at most
  int64_t p = slots <= 2048 ? 1 : ceil_div(slots, 1024);
  if (p > 148) p = 148;
  *per_part = (int)(ceil_div(ceil_div(slots, p), 256) * 256);
  if (*per_part == 0) *per_part = 256;
  *parts = (int)ceil_div(slots, *per_part);
  if (*parts == 0) *parts = 1;
}

}  // namespace altob200

using namespace altob200;

static bool route_type_ok(int32_t dtype) { return dtype == ALTOB200_DT_BF16 || dtype == ALTOB200_DT_F32; }

#define ROUTE_BY_V(LAUNCH, B)                 \
  do {                                        \
    if (E <= 32) LAUNCH(B, 1);                \
    else if (E <= 64) LAUNCH(B, 2);           \
    else if (E <= 128) LAUNCH(B, 4);          \
    else if (E <= 256) LAUNCH(B, 8);          \
    else LAUNCH(B, 16);                       \
  } while (0)

extern "C" int altob200_route_forward(const altob200_route_params* p, const void* logits, int64_t tokens, int64_t ld,
                                      const float* bias, int32_t* ids, float* weights, void* stream) {
  if (p == nullptr || tokens < 0 || p->experts <= 0 || p->top_k <= 0) return ALTOB200_EINVAL_SHAPE;
  if (!route_type_ok(p->dtype)) return ALTOB200_EUNSUPPORTED;
  if (p->experts > ROUTE_MAX_E || p->top_k > ROUTE_MAX_K || p->num_groups > ROUTE_MAX_GROUPS) return ALTOB200_ELIMIT;
  if (p->num_groups <= 0 || p->experts % p->num_groups != 0 || p->groups_kept <= 0 || p->groups_kept > p->num_groups ||
      (p->group_top != 1 && p->group_top != 2) || p->top_k > p->groups_kept * (p->experts / p->num_groups))
    return ALTOB200_EINVAL_SHAPE;
  if (tokens == 0) return ALTOB200_OK;
  if (logits == nullptr || ids == nullptr || weights == nullptr || ld < p->experts) return ALTOB200_EINVAL_SHAPE;
  RouteArgs a;
  a.logits = logits; a.bias = bias; a.ids = ids; a.weights = weights; a.tokens = tokens; a.ld = ld;
  a.experts = p->experts; a.k = p->top_k; a.sigmoid = p->sigmoid; a.groups = p->num_groups; a.kept = p->groups_kept;
  // groups that are all kept, or judged by their best expert without a bias, need no computed keys
  a.group_top = p->num_groups > 1 && p->groups_kept < p->num_groups ? p->group_top : 1;
  if (p->groups_kept == p->num_groups) a.groups = a.kept = 1;
  a.renorm = p->renormalize; a.scale = p->scale;
  const int E = p->experts;
  const size_t smem = a.groups > 1 ? (size_t)8 * (E + a.groups) * 8 : 0;
  int64_t blocks = ceil_div(tokens, 8);
  if (blocks > 148 * 8) blocks = 148 * 8;
#define RUN(B, V) (void)launch_after(route_forward_kernel<B, V>, dim3((unsigned)blocks), dim3(256), smem, (cudaStream_t)stream, a)
  if (p->dtype == ALTOB200_DT_BF16) ROUTE_BY_V(RUN, true);
  else ROUTE_BY_V(RUN, false);
#undef RUN
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

extern "C" int altob200_route_backward(const altob200_route_params* p, const void* logits, int64_t tokens, int64_t ld,
                                       const int32_t* ids, const float* grad_weights, void* grad_logits, void* stream) {
  if (p == nullptr || tokens < 0 || p->experts <= 0 || p->top_k <= 0) return ALTOB200_EINVAL_SHAPE;
  if (!route_type_ok(p->dtype)) return ALTOB200_EUNSUPPORTED;
  if (p->experts > ROUTE_MAX_E || p->top_k > ROUTE_MAX_K) return ALTOB200_ELIMIT;
  if (tokens == 0) return ALTOB200_OK;
  if (logits == nullptr || ids == nullptr || grad_weights == nullptr || grad_logits == nullptr || ld < p->experts)
    return ALTOB200_EINVAL_SHAPE;
  RouteGradArgs a;
  a.logits = logits; a.ids = ids; a.grad = grad_weights; a.grad_logits = grad_logits; a.tokens = tokens; a.ld = ld;
  a.experts = p->experts; a.k = p->top_k; a.sigmoid = p->sigmoid; a.renorm = p->renormalize; a.scale = p->scale;
  const int E = p->experts;
  int64_t blocks = ceil_div(tokens, 8);
  if (blocks > 148 * 8) blocks = 148 * 8;
#define RUN(B, V) (void)launch_after(route_backward_kernel<B, V>, dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, a)
  if (p->dtype == ALTOB200_DT_BF16) ROUTE_BY_V(RUN, true);
  else ROUTE_BY_V(RUN, false);
#undef RUN
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

extern "C" int64_t altob200_expert_plan_work_bytes(int64_t slots, int32_t experts) {
  if (slots <= 0 || experts <= 0) return 0;
  int parts, per_part;
  plan_split(slots, &parts, &per_part);
  return parts > 1 ? (int64_t)parts * experts * 4 : 0;
}

extern "C" int altob200_expert_plan(const void* ids, int32_t ids_bits, int64_t tokens, int32_t k, int32_t experts,
                                    int32_t align, int64_t rows, int32_t* token, int32_t* position, int32_t* slot,
                                    int32_t* offs, int32_t* counts, void* work, void* stream) {
  if (tokens < 0 || k <= 0 || experts <= 0 || align <= 0 || rows < 0) return ALTOB200_EINVAL_SHAPE;
  if (ids_bits != 32 && ids_bits != 64) return ALTOB200_EUNSUPPORTED;
  const int64_t slots = tokens * k;
  if (experts > PLAN_MAX_E || tokens > (1ll << 31) / k || slots + (int64_t)experts * align >= (1ll << 31) - 1 || rows >= (1ll << 31) - 1) return ALTOB200_ELIMIT;
  if ((slots > 0 && (ids == nullptr || slot == nullptr)) || (rows > 0 && (token == nullptr || position == nullptr)) ||
      offs == nullptr || counts == nullptr)
    return ALTOB200_EINVAL_SHAPE;
  PlanArgs a;
  a.ids = ids; a.token = token; a.position = position; a.slot = slot; a.offs = offs; a.counts = counts;
  a.hist = reinterpret_cast<int32_t*>(work);
  a.slots = slots; a.rows = rows; a.k = k; a.experts = experts; a.align = align; a.wide = ids_bits == 64;
  plan_split(slots, &a.parts, &a.per_part);
  if (a.parts > 1 && work == nullptr) return ALTOB200_EINVAL_SHAPE;
  const cudaStream_t st = (cudaStream_t)stream;
  if (a.parts > 1) (void)launch_after(plan_count_kernel, dim3(a.parts), dim3(256), (size_t)experts * 4, st, a);
  (void)launch_after(plan_place_kernel, dim3(a.parts), dim3(256), (size_t)experts * 11 * 4, st, a);
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}
