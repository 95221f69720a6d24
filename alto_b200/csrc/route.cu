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
#include <type_traits>

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
  int32_t computed;          // keys are scores (and bias), not the logits
  int32_t checked;           // keys in fp32 words do not settle every decision
  int32_t per;               // experts a lane holds
  int32_t lanes_per_group;   // that hold a group, a power of two; 0: groups are not made of whole lanes so
  int32_t scratch;           // doubles of shared memory a warp has
  float score_room;          // how far two scores are off together, relative
};

static constexpr int ROUTE_MAX_K = 16, ROUTE_MAX_E = 512, ROUTE_MAX_GROUPS = 32;   // a choice and its successor fit a warp
static constexpr unsigned FULL = 0xFFFFFFFFu;

template <bool BF16>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
  if constexpr (BF16) return __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(p) + i));
  else return __ldg(reinterpret_cast<const float*>(p) + i);
}

// Unsigned words in the order of the floats; a (positive) NaN above everything, 0 below everything.
__device__ __forceinline__ uint32_t ordered_bits(uint32_t b) { return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u); }
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  if (v != v) return ~0ull;
  return (b >> 63) ? ~b : (b | (1ull << 63));
}
template <int LANES = 32>
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}
template <class F, int LANES = 32>
__device__ __forceinline__ F warp_add(F v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ float from_ordered(uint32_t w) { return u2f(w >> 31 ? w & 0x7FFFFFFFu : ~w); }
// The key of a word whose LOW bits hold something else: the key itself or up to LOW steps below it.  -inf is the one number
// whose own low bits are ones; without them its word would be a NaN's.
template <uint32_t LOW>
__device__ __forceinline__ float key_of_word(uint32_t w) {
  return (w | LOW) == 0x007FFFFFu ? -INFINITY : from_ordered(w & ~LOW);
}

__device__ __forceinline__ uint64_t warp_max_key(uint64_t v) {
  const uint32_t hi = __reduce_max_sync(FULL, (uint32_t)(v >> 32));
  const uint32_t lo = __reduce_max_sync(FULL, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
  return ((uint64_t)hi << 32) | lo;
}

// The choice of one token by one warp in double: what the fp32 form hands over because two keys are too near.  Lane l looks
// after experts l, l + 32, ...; `keys` is the warp's shared memory, [experts].  Lane i < k returns the i-th choice.
template <bool BF16>
__device__ __forceinline__ int choose_in_double(const RouteArgs& a, int64_t row, double* keys) {
  const int lane = threadIdx.x & 31, E = a.experts, size = E / a.groups;
  double m = -INFINITY, z = 0.0;
  if (a.computed && !a.sigmoid) {
    for (int e = lane; e < E; e += 32) m = fmax(m, (double)logit_at<BF16>(a.logits, row + e));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(FULL, m, o));
    for (int e = lane; e < E; e += 32) z += exp((double)logit_at<BF16>(a.logits, row + e) - m);
    z = warp_add(z);
  }
  __syncwarp();
  for (int e = lane; e < E; e += 32) {
    const double l = logit_at<BF16>(a.logits, row + e), s = !a.computed ? l + 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - m) / z;
    keys[e] = a.bias != nullptr ? s + (double)__ldg(a.bias + e) : s;
  }
  __syncwarp();
  uint32_t allowed = FULL;   // bit g: group g
  if (a.groups > 1) {
    uint64_t best = 0, second = 0;
    int every = 1;             // lanes that look after a group
    while (every * 2 * a.groups <= 32) every *= 2;
    const int group = lane / every;
    const auto meet = [&](uint64_t b2, uint64_t s2) {
      const uint64_t low = best < b2 ? best : b2, high = second > s2 ? second : s2;
      second = low > high ? low : high;
      best = best > b2 ? best : b2;
    };
    if (group < a.groups)
      for (int i = lane & (every - 1); i < size; i += every) meet(ordered(keys[group * size + i]), 0ull);
    for (int o = 1; o < every; o <<= 1) meet(__shfl_xor_sync(FULL, best, o), __shfl_xor_sync(FULL, second, o));
    const auto value = [](uint64_t w) { return __longlong_as_double((long long)(w >> 63 ? w & ~(1ull << 63) : ~w)); };
    const uint64_t word = group >= a.groups ? 0 : a.group_top == 2 && size > 1 ? ordered(value(best) + value(second)) : best;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint64_t other = __shfl_sync(FULL, word, g * every);
      rank += other > word || (other == word && g < group) ? 1 : 0;
    }
    allowed = 0u;
    for (int g = 0; g < a.groups; ++g) allowed |= (uint32_t)__shfl_sync(FULL, rank < a.kept ? 1 : 0, g * every) << g;
  }
  int mine = 0;
  uint64_t last = ~0ull;     // the previous choice: what comes next is smaller, or equal at a higher index
  int last_e = -1;
  for (int i = 0; i < a.k; ++i) {
    uint64_t top = 0;
    int where = 0x7FFFFFFF;
    for (int e = lane; e < E; e += 32) {
      const uint64_t w = (allowed >> (a.groups > 1 ? e / size : 0)) & 1u ? ordered(keys[e]) : 0ull;
      if ((w < last || (w == last && e > last_e)) && w > top) {
        top = w;
        where = e;
      }
    }
    last = warp_max_key(top);
    last_e = (int)__reduce_min_sync(FULL, top == last ? (uint32_t)where : 0x7FFFFFFFu);
    if (lane == i) mine = last_e;
  }
  return mine;
}

// Descending order of N registers from LO on (Batcher's odd-even merge sort).
__device__ __forceinline__ void exchange(uint32_t& u, uint32_t& v) {
  const uint32_t big = max(u, v);
  v = min(u, v);
  u = big;
}
template <int LO, int N, int R>
__device__ __forceinline__ void merge_words(uint32_t* w) {
  if constexpr (2 * R < N) {
    merge_words<LO, N, 2 * R>(w);
    merge_words<LO + R, N, 2 * R>(w);
#pragma unroll
    for (int i = LO + R; i + R < LO + N; i += 2 * R) exchange(w[i], w[i + R]);
  } else {
    exchange(w[LO], w[LO + R]);
  }
}
template <int LO, int N>
__device__ __forceinline__ void sort_words(uint32_t* w) {
  if constexpr (N > 1) {
    sort_words<LO, N / 2>(w);
    sort_words<LO + N / 2, N / 2>(w);
    merge_words<LO, N, 1>(w);
  }
}

// Keys of a lane's experts in fp32 (the logits, or scores and bias), and the largest score that the token can have.  Every
// key comes out of an addition, whose NaN is the positive one: its bits are above everything.
template <int V>
__device__ __forceinline__ float keys_of(const RouteArgs& a, const float* l, const float* b, float* key) {
  if (!a.computed) {
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = l[j] + 0.0f;   // -0 is 0
    return 0.0f;
  }
  float r = 1.0f;
  if (a.sigmoid) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(key[j]) : "f"(1.0f + fast_exp(fminf(fmaxf(-l[j], -126.0f), 126.0f))));
      if (l[j] != l[j]) key[j] = l[j];
    }
  } else {
    float m = l[0], z = 0.0f;
#pragma unroll
    for (int j = 1; j < V; ++j) m = fmaxf(m, l[j]);
    m = warp_max(m);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = l[j] - m;
      key[j] = d >= -126.0f ? fast_exp(d) : d != d ? d : 0.0f;
      z += key[j];
    }
    r = 1.0f / warp_add(z);
  }
#pragma unroll
  for (int j = 0; j < V; ++j) key[j] = key[j] * r + b[j];
  return r;
}

// The choice of one token by one warp in fp32; lane l holds the a.per experts from l * a.per on.  Lane i < k returns the i-th
// choice and its logit.  *sure: every decision holds in exact arithmetic too.
//
// A key is held as an ordered word whose lowest bits are V - 1 - j: each lane sorts its V words once, a choice is then the
// largest of the lanes' first words, and its lane moves its list up.  Words are compared across lanes without those bits
// and the lowest lane is taken, so equal keys come out by expert.  The bits that j takes are missing from every
// comparison (none of a bf16 logit's), which `room` allows for below; they are zero again in every key that a margin is taken
// of (with j left in them two keys could move by V - 1 steps each, in opposite directions).
template <bool BF16, int V, bool WHOLE>
__device__ __forceinline__ int choose(const RouteArgs& a, int64_t row, const float* l, const float* b, uint32_t* words,
                                      float* logit, bool* sure) {
  constexpr uint32_t LOW = V - 1;
  // two keys that differ by less may be in the other order: what is cut off the lower one, and half a step of each sum
  constexpr float CUT = (V - 1) * 1.1920929e-7f + 1.2e-7f;
  constexpr float TINY = 2.4e-38f;   // two scores below the least normal number, which are zero here
  const int lane = threadIdx.x & 31, per = WHOLE ? V : a.per;
  uint32_t word[V];
  *sure = true;
  float most;
  {
    float key[V];
    most = keys_of<V>(a, l, b, key);
#pragma unroll
    for (int j = 0; j < V; ++j) word[j] = ordered_bits(f2u(key[j]));
  }
#pragma unroll
  for (int j = 0; j < V; ++j)
    word[j] = WHOLE || (j < per && lane * per + j < a.experts) ? (word[j] & ~LOW) | (LOW - (uint32_t)j) : 0u;
  int left = a.experts;
  uint32_t kept = 1u;   // bit g (times the lanes of a group): group g
  if (a.groups > 1) {
    // a group's two best: by the lanes that hold it, or, where groups do not consist of a power of two of whole lanes,
    // by one lane from shared memory
    const int size = a.experts / a.groups, every = a.lanes_per_group > 0 ? a.lanes_per_group : 1, mine = lane / every;
    uint32_t best = 0u, second = 0u;
    if (a.lanes_per_group > 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        second = max(second, min(best, word[j]));
        best = max(best, word[j]);
      }
      for (int o = 1; o < every; o <<= 1) {
        const uint32_t b2 = __shfl_xor_sync(FULL, best, o), s2 = __shfl_xor_sync(FULL, second, o);
        second = max(max(second, s2), min(best, b2));
        best = max(best, b2);
      }
    } else {
      __syncwarp();
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j < per && lane * per + j < a.experts) words[lane * per + j + (lane * per + j) / size] = word[j];
      __syncwarp();
      if (mine < a.groups)
        for (int i = 0; i < size; ++i) {
          const uint32_t w = words[mine * (size + 1) + i];   // a word between groups: their lanes read different banks
          second = max(second, min(best, w));
          best = max(best, w);
        }
    }
    const bool two = a.group_top == 2 && size > 1;
    const float first = key_of_word<LOW>(best), other = two ? key_of_word<LOW>(second) : 0.0f, of_group = first + other;
    // the kept groups one by one, the lowest among equals
    uint32_t rest = mine >= a.groups ? 0u : a.group_top == 2 ? ordered_bits(f2u(of_group)) : best & ~LOW;
    kept = 0u;
    for (int i = 0; i < a.kept; ++i) {
      const uint32_t top = __reduce_max_sync(FULL, rest);
      const int last = __ffs(__ballot_sync(FULL, rest == top)) - 1;
      kept |= 1u << last;
      if (mine * every == last) rest = 0u;
    }
    if (a.checked) {
      // Each group's own margin (half a step of the sum and one of the margin's own sum on top of CUT), so that a group far
      // below the decision, as one masked by a large negative bias is, widens nobody else's: every kept sum as low as it
      // can be is above every other as high as it can be.  Infinities have no margin; equal ones are not told apart here.
      const float margin = fabsf(of_group) < INFINITY ? a.score_room * most + (CUT + 2.4e-7f) * (fabsf(first) + fabsf(other)) + TINY : 0.0f;
      const bool in = (kept >> (mine * every)) & 1u;
      const uint32_t low = __reduce_min_sync(FULL, mine < a.groups && in ? ordered_bits(f2u(of_group - margin)) : FULL);
      const uint32_t high = __reduce_max_sync(FULL, mine < a.groups && !in ? ordered_bits(f2u(of_group + margin)) : 0u);
      if (low <= high) *sure = false;
    }
    left = a.kept * size;
    if (a.lanes_per_group > 0) {
      const bool in = (kept >> (mine * every)) & 1u;
#pragma unroll
      for (int j = 0; j < V; ++j) word[j] = in ? word[j] : 0u;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (!((kept >> (((lane * per + j) / size) & 31)) & 1u)) word[j] = 0u;
    }
  }
  sort_words<0, V>(word);
  // the next one after the last is looked at too, where there is one
  const int picks = a.checked && left > a.k ? a.k + 1 : a.k;
  int mine = 0;
  uint32_t mine_word = 0u;
  for (int i = 0; i < picks; ++i) {
    const uint32_t best = __reduce_max_sync(FULL, word[0] & ~LOW);
    const int owner = __ffs(__ballot_sync(FULL, (word[0] & ~LOW) == best)) - 1;
    const uint32_t taken = V > 1 ? __shfl_sync(FULL, word[0], owner) : best;
    const bool up = lane == owner;
#pragma unroll
    for (int j = 0; j + 1 < V; ++j) word[j] = up ? word[j + 1] : word[j];
    word[V - 1] = up ? 0u : word[V - 1];
    if (lane == i) {
      mine = owner * per + (int)(LOW - (taken & LOW));
      mine_word = taken;
    }
  }
  const bool on = lane < picks;
  const float my_l = on ? logit_at<BF16>(a.logits, row + mine) : 0.0f;
  *logit = my_l;
  if (a.checked) {
    // Neighbours in the order whose keys fp32 cannot tell apart, unless their inputs are the same.  A softmax is off by at
    // most 7e-6 of itself (the rounding of l - m before the exponential, up to 88 * 2^-24, is the most of it), a sigmoid by
    // 6e-7.
    const float my_b = on && a.bias != nullptr ? __ldg(a.bias + mine) : 0.0f, my_key = key_of_word<LOW>(mine_word);
    const float next_l = __shfl_down_sync(FULL, my_l, 1), next_b = __shfl_down_sync(FULL, my_b, 1);
    const float next_key = __shfl_down_sync(FULL, my_key, 1);
    const float cut = CUT * fmaxf(fabsf(my_key), fabsf(next_key)) + TINY, gap = my_key - next_key;
    const float room = a.score_room * fmaxf(my_key - my_b, next_key - next_b) + cut;
    if (__any_sync(FULL, lane + 1 < a.k && gap <= room && !(my_l == next_l && my_b == next_b))) *sure = false;
    // The last choice against everything that is left: all of it is below the next one, but with a bias any of it may have
    // a larger score, and error, than that.
    const bool far = gap > (a.bias != nullptr ? a.score_room * most + cut : room);
    if (*sure && picks > a.k && !__shfl_sync(FULL, far, a.k - 1)) {
      const float last_l = __shfl_sync(FULL, my_l, a.k - 1), last_b = __shfl_sync(FULL, my_b, a.k - 1);
      const float last_key = __shfl_sync(FULL, my_key, a.k - 1);
      const float low = last_key - a.score_room * (last_key - last_b) - CUT * fabsf(last_key) - TINY;
      float key[V];
      keys_of<V>(a, l, b, key);
      bool over = false;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = lane * per + j;
        bool out = (WHOLE || (j < per && e < a.experts)) && !(l[j] == last_l && b[j] == last_b);
        if (a.groups > 1) {
          const int at = a.lanes_per_group > 0 ? lane / a.lanes_per_group * a.lanes_per_group : e / (a.experts / a.groups);
          out = out && ((kept >> (at & 31)) & 1u);
        }
        for (int i = 0; i < a.k; ++i) {
          const int taken = __shfl_sync(FULL, mine, i);   // by every lane
          out = out && taken != e;
        }
        over = over || (out && key[j] + a.score_room * (key[j] - b[j]) + CUT * fabsf(key[j]) >= low);
      }
      if (__any_sync(FULL, over)) *sure = false;
    }
  }
  return mine;
}

// A lane's V consecutive logits from p on, aligned to a vector of them.
template <bool BF16, int V>
__device__ __forceinline__ void load_logits(const void* logits, int64_t at, float* l) {
  constexpr int BYTES = V * (BF16 ? 2 : 4), WORDS = BYTES / 4;
  if constexpr (BYTES < 4) {
    l[0] = logit_at<BF16>(logits, at);
  } else {
    const char* p = reinterpret_cast<const char*>(logits) + at * (BF16 ? 2 : 4);
    uint32_t w[WORDS];
    if constexpr (BYTES == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (BYTES == 8) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
      for (int q = 0; q < WORDS / 4; ++q) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + q);
        w[4 * q] = v.x; w[4 * q + 1] = v.y; w[4 * q + 2] = v.z; w[4 * q + 3] = v.w;
      }
    }
#pragma unroll
    for (int q = 0; q < WORDS; ++q) {
      if constexpr (BF16) {
        l[2 * q] = bf16lo_to_f32(w[q]);
        l[2 * q + 1] = bf16hi_to_f32(w[q]);
      } else {
        l[q] = u2f(w[q]);
      }
    }
  }
}

// Weights of the chosen, on lanes i < k (l: the chosen logit).  `m`, `z`: maximum and sum of exponentials
// over all experts, used by the softmax that is not renormalised.  Ratios are formed from the chosen alone, so that they
// hold however small the scores are; a token whose chosen scores are all zero gets zero weights.
template <int LANES = 32>
__device__ __forceinline__ float chosen_weight(bool on, float l, int sigmoid, int renorm, float m, float z, float* total) {
  *total = 1.0f;
  if (sigmoid) {
    // e^(l - c) / (1 + e^l) with c = min(0, the largest chosen logit): in range for any logits
    float c = 0.0f;
    if (renorm) {
      c = fminf(warp_max<LANES>(on ? l : -INFINITY), 0.0f);
      if (c == -INFINITY) c = 0.0f;
    }
    const float num = l > 0.0f ? 1.0f : fast_exp(fmaxf(l - c, -126.0f)), den = 1.0f + fast_exp(fmaxf(-fabsf(l), -126.0f));
    const float s = !on ? 0.0f : l != l ? l : __fdividef(num, den);
    if (!renorm) return s;
    *total = warp_add<float, LANES>(s);
    return *total == 0.0f ? 0.0f : __fdiv_rn(s, *total);   // a choice of one has weight 1, and no gradient
  }
  if (!renorm) {
    const float d = l - m;
    return on && m != -INFINITY ? __fdiv_rn(d >= -126.0f ? fast_exp(d) : d != d ? d : 0.0f, z) : 0.0f;
  }
  const float top = warp_max<LANES>(on ? l : -INFINITY);
  const float d = l - top, s = !on ? 0.0f : d >= -126.0f ? fast_exp(d) : d != d ? d : 0.0f;
  *total = warp_add<float, LANES>(s);   // a NaN where top = -inf, and where there is one
  if (top == -INFINITY && !(l != l)) return 0.0f;
  return __fdiv_rn(s, *total);
}

// Weights of a token whose choice is made: lane i < k holds the i-th chosen expert and its logit.
template <int V>
__device__ __forceinline__ void write_choice(const RouteArgs& a, int64_t t, const float* l, int chosen, float mine) {
  const int lane = threadIdx.x & 31;
  const bool on = lane < a.k;
  float m = 0.0f, z = 1.0f, total;
  if (!a.sigmoid && !a.renorm) {
    m = l[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = fmaxf(m, l[j]);
    m = warp_max(m);
    z = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = l[j] - m;   // -inf for experts that are not there; m = -inf is seen to by chosen_weight
      z += d >= -126.0f ? fast_exp(d) : d != d ? d : 0.0f;
    }
    z = warp_add(z);
  }
  float w = chosen_weight(on, mine, a.sigmoid, a.renorm, m, z, &total);
  if (a.computed && !a.sigmoid) {   // a NaN that is not among the chosen makes every score one all the same
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

// A warp takes 32 tokens at most (the launch sees to it), so that those whose choice is not certain in fp32 are bits of a
// word; they are done in double behind the others, by a loop that the registers of the first do not have to make room for.
template <bool BF16, int V, bool WHOLE>
__global__ void __launch_bounds__(256) route_forward_kernel(RouteArgs a) {
  extern __shared__ double route_smem[];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  double* const scratch = route_smem + (threadIdx.x >> 5) * a.scratch;
  const int per = WHOLE ? V : a.per;
  float b[V];
#pragma unroll
  for (int j = 0; j < V; ++j) b[j] = a.bias != nullptr && j < per && lane * per + j < a.experts ? __ldg(a.bias + lane * per + j) : 0.0f;
  const auto load = [&](int64_t row, float* l) {
    if constexpr (WHOLE) {
      load_logits<BF16, V>(a.logits, row + lane * V, l);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) l[j] = j < per && lane * per + j < a.experts ? logit_at<BF16>(a.logits, row + lane * per + j) : -INFINITY;
    }
  };
  const int64_t first = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), step = (int64_t)gridDim.x * 8;
  uint32_t again = 0u, bit = 1u;
  for (int64_t t = first; t < a.tokens; t += step, bit <<= 1) {
    float l[V], mine;
    load(t * a.ld, l);
    bool sure;
    const int chosen = choose<BF16, V, WHOLE>(a, t * a.ld, l, b, reinterpret_cast<uint32_t*>(scratch), &mine, &sure);
    if (sure) write_choice<V>(a, t, l, chosen, mine);
    else again |= bit;
  }
  while (again != 0u) {
    const int64_t t = first + (__ffs(again) - 1) * step;
    again &= again - 1u;
    const int chosen = choose_in_double<BF16>(a, t * a.ld, scratch);
    float l[V];
    load(t * a.ld, l);
    write_choice<V>(a, t, l, chosen, lane < a.k ? logit_at<BF16>(a.logits, t * a.ld + chosen) : 0.0f);
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
  int32_t vector;        // rows of grad_logits allow 16-byte stores
};

//   softmax              dl_e = scale p_e (g_e [chosen] - sum g p)       with p over all experts, or over the chosen when
//                                                                        renormalised (then zero for the others)
//   sigmoid              dl_i = scale s_i (1 - s_i) g_i
//   sigmoid, renormalised dl_i = scale q_i (1 - s_i) (g_i - sum g q)     q = s / sum s
//
// Where only the chosen have a gradient (all but the first): 16 lanes a token write its row of zeros, and over it, once
// they have all written, the k values.  65536 x 256 fp32: 67 MB of zeros, 10 us at the copy rate.
template <bool BF16>
__global__ void __launch_bounds__(256) route_backward_chosen_kernel(RouteGradArgs a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, float>::type;
  grid_dependency_wait();
  const int lane = threadIdx.x & 15;
  const int64_t step = (int64_t)gridDim.x * 16;
  // both halves of a warp go round together (shuffles); one behind the last token does nothing
  const int64_t mine = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), warp_first = mine & ~1ll;
  for (int64_t lead = warp_first, t = mine; lead < a.tokens; lead += step, t += step) {
    const bool live = t < a.tokens;
    T* const out = reinterpret_cast<T*>(a.grad_logits) + t * a.experts;
    int id = live && lane < a.k ? __ldg(a.ids + t * a.k + lane) : -1;
    if (id >= a.experts) id = -1;
    const bool on = id >= 0;
    const float g = on ? __ldg(a.grad + t * a.k + lane) : 0.0f;
    const float l = on ? logit_at<BF16>(a.logits, t * a.ld + id) : 0.0f;
    if (live) {
      if (a.vector) {
        for (int c = lane; c < a.experts * (int)sizeof(T) / 16; c += 16) reinterpret_cast<uint4*>(out)[c] = make_uint4(0u, 0u, 0u, 0u);
      } else {
        for (int e = lane; e < a.experts; e += 16) out[e] = (T)0.0f;
      }
    }
    float total;
    const float w = chosen_weight<16>(on, l, a.sigmoid, a.renorm, 0.0f, 1.0f, &total);
    const float sum = a.renorm ? warp_add<float, 16>(on ? g * w : 0.0f) : 0.0f;
    const float rest = a.sigmoid ? 1.0f / (1.0f + expf(l)) : 1.0f;   // 1 - s
    const float d = a.scale * w * rest * (g - sum);
    __syncwarp();
    if (on) out[id] = (T)d;
    __syncwarp();
  }
}

// The softmax over all experts: every expert has a gradient.
template <bool BF16, int V>
__global__ void __launch_bounds__(256) route_backward_kernel(RouteGradArgs a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, float>::type;
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < a.tokens; t += (int64_t)gridDim.x * 8) {
    const int64_t row = t * a.ld;
    int id = lane < a.k ? __ldg(a.ids + t * a.k + lane) : -1;
    if (id >= a.experts) id = -1;
    const bool on = id >= 0;
    const float l = on ? logit_at<BF16>(a.logits, row + id) : 0.0f, g = on ? __ldg(a.grad + t * a.k + lane) : 0.0f;
    float m = -INFINITY, z = 0.0f, total, all[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      all[j] = lane + 32 * j < a.experts ? logit_at<BF16>(a.logits, row + lane + 32 * j) : -INFINITY;
      m = fmaxf(m, all[j]);
    }
    m = warp_max(m);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float d = all[j] - m;   // experts that are not there are -inf; m = -inf is seen to below
      all[j] = d >= -126.0f ? fast_exp(d) : d != d ? d : 0.0f;
      z += all[j];
    }
    z = warp_add(z);
    const float w = chosen_weight(on, l, 0, 0, m, z, &total);
    const float sum = warp_add(on ? g * w : 0.0f), of_all = m != -INFINITY ? -a.scale * sum / z : 0.0f;
    // the terms that every expert has, and over them, once the warp has written those, the chosen
    T* const out = reinterpret_cast<T*>(a.grad_logits) + t * a.experts;
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (lane + 32 * j < a.experts) out[lane + 32 * j] = (T)(m != -INFINITY ? of_all * all[j] : 0.0f);
    __syncwarp();
    if (on) out[id] = (T)(a.scale * w * (g - sum));
    __syncwarp();
  }
}

// ---------------------------------------------------------------------------------------
// Row plan: a counting sort of the routed slots by expert, stable, every expert's run padded to `align` rows.
//
// The slots are cut into parts, one per CTA and 32 x (1 to 8) per warp, held in registers.  Counting: every part's slots
// by expert.  Placing: a CTA adds up the parts in front of its own (and all, for the runs' starts), counts its warps'
// slots, and a slot's row is start + parts before + warps before + lanes of the same expert before (match.any).  Integers
// only, so no order changes the result.  One part needs no counting launch; more than PLAN_DIRECT parts get a launch in
// between that sums over parts, so that the work stays linear.  What bounds it is latency, dependent round
// trips to L2 and shared memory, and two launches: 65 536 slots over 32 experts 8.0 us in a stream, 262 144 over 256 14.0
// (20 us a call with the host's five allocations and two launches; tensor operations 290 and 297).
// ---------------------------------------------------------------------------------------
struct PlanArgs {
  const void* ids;       // [slots] int32 or int64
  int32_t* token;        // [rows] token of a row, -1: padding
  int32_t* position;     // [rows] routed slot of a row, -1: padding
  int32_t* slot;         // [slots] row of a routed slot, -1: no row
  int32_t* offs;         // [experts] ends of the padded runs
  int32_t* counts;       // [experts] rows without padding
  int32_t* hist;         // [parts][experts], and behind it the sums [experts]; unused with one part
  int64_t slots, rows;
  int32_t k, experts, align, wide, parts, each;   // each: slots a lane has, so a part is warps * 32 * each
};
static constexpr int PLAN_MAX_E = 1024, PLAN_EACH = 8, PLAN_DIRECT = 128;

__device__ __forceinline__ int plan_id(const PlanArgs& a, int64_t i) {
  if (a.wide) {
    const int64_t v = __ldg(reinterpret_cast<const long long*>(a.ids) + i);
    return v >= 0 && v < a.experts ? (int)v : -1;
  }
  const int v = __ldg(reinterpret_cast<const int32_t*>(a.ids) + i);
  return v >= 0 && v < a.experts ? v : -1;
}
// rows of a run, padding included
__device__ __forceinline__ int plan_run(int count, int align) { return count == 0 ? align : (count + align - 1) / align * align; }

__global__ void __launch_bounds__(512) plan_count_kernel(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  grid_dependency_wait();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) plan_smem[e] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * blockDim.x * a.each + threadIdx.x;
  int id[PLAN_EACH];
#pragma unroll
  for (int j = 0; j < PLAN_EACH; ++j) {
    const int64_t i = first + (int64_t)j * blockDim.x;
    id[j] = j < a.each && i < a.slots ? plan_id(a, i) : -1;
  }
#pragma unroll
  for (int j = 0; j < PLAN_EACH; ++j)
    if (id[j] >= 0) atomicAdd(&plan_smem[id[j]], 1);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.hist[(int64_t)blockIdx.x * a.experts + e] = plan_smem[e];
}

// hist[p][e] <- sum of the parts in front of p; the totals behind it.  32 experts a CTA, its warps over slices of the parts.
__global__ void __launch_bounds__(1024) plan_sum_kernel(PlanArgs a) {
  __shared__ int32_t of[32][33];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  const int slice = (a.parts + 31) / 32, first = warp * slice, stop = min(first + slice, a.parts);
  int sum = 0;
  if (e < a.experts) {
#pragma unroll 8
    for (int p = first; p < stop; ++p) sum += a.hist[(int64_t)p * a.experts + e];
  }
  of[warp][lane] = sum;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < warp; ++w) before += of[w][lane];
  if (e >= a.experts) return;
  for (int p = first; p < stop; ++p) {
    int32_t* at = a.hist + (int64_t)p * a.experts + e;
    const int c = *at;
    *at = before;
    before += c;
  }
  if (warp == 31) a.hist[(int64_t)a.parts * a.experts + e] = before;
}

__global__ void __launch_bounds__(512) plan_place_kernel(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5, E = a.experts;
  int32_t* const of_warp = plan_smem;                       // [warps][E] counts of the warps, then next rows
  int32_t* const count = plan_smem + warps * E;             // [E] rows of an expert
  int32_t* const start = count + E;                         // [E] its first row
  int32_t* const before = start + E;                        // [E] rows from earlier parts
  __shared__ int32_t scan[32];
  grid_dependency_wait();
  const int64_t first = ((int64_t)blockIdx.x * warps + warp) * 32 * a.each + lane;
  int id[PLAN_EACH];
#pragma unroll
  for (int j = 0; j < PLAN_EACH; ++j) id[j] = j < a.each && first + 32 * j < a.slots ? plan_id(a, first + 32 * j) : -1;
  for (int i = tid; i < (warps + 3) * E; i += threads) plan_smem[i] = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PLAN_EACH; ++j)
    if (id[j] >= 0) atomicAdd(&of_warp[warp * E + id[j]], 1);
  // totals and earlier parts, by expert: as many threads an expert as there are
  if (a.parts > PLAN_DIRECT) {
    for (int e = tid; e < E; e += threads) {
      count[e] = a.hist[(int64_t)a.parts * E + e];
      before[e] = a.hist[(int64_t)blockIdx.x * E + e];
    }
  } else if (a.parts > 1) {
    int wide = 32;
    while (wide < E && wide < threads) wide *= 2;
    const int slices = threads / wide;
    for (int e = tid & (wide - 1); e < E; e += wide) {
      int all = 0, earlier = 0;
#pragma unroll 16
      for (int p = tid / wide; p < a.parts; p += slices) {
        const int c = a.hist[(int64_t)p * E + e];
        all += c;
        earlier += p < (int)blockIdx.x ? c : 0;
      }
      atomicAdd(&count[e], all);
      atomicAdd(&before[e], earlier);
    }
  }
  __syncthreads();
  if (a.parts == 1) {
    for (int e = tid; e < E; e += threads) {
      int all = 0;
      for (int w = 0; w < warps; ++w) all += of_warp[w * E + e];
      count[e] = all;
    }
    __syncthreads();
  }
  // first rows: an exclusive sum of the runs, E / threads (rounded up) neighbouring experts a thread
  const int per = (E + threads - 1) / threads;
  int mine = 0;
  for (int j = 0; j < per; ++j)
    if (tid * per + j < E) mine += plan_run(count[tid * per + j], a.align);
  int sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(FULL, sum, o);
    if (lane >= o) sum += v;
  }
  if (lane == 31) scan[warp] = sum;
  __syncthreads();
  int at = sum - mine;
  for (int w = 0; w < warp; ++w) at += scan[w];
  for (int j = 0; j < per; ++j) {
    const int e = tid * per + j;
    if (e < E) {
      start[e] = at;
      int row = at + before[e];
      at += plan_run(count[e], a.align);
      if (blockIdx.x == 0) {
        a.offs[e] = at;
        a.counts[e] = count[e];
      }
      for (int w = 0; w < warps; ++w) {   // next row of every (warp, expert)
        const int c = of_warp[w * E + e];
        of_warp[w * E + e] = row;
        row += c;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PLAN_EACH; ++j) {
    if (j >= a.each) break;
    const int64_t i = first + 32 * j;
    const int e = id[j];
    const unsigned same = __match_any_sync(FULL, e);
    int row = -1;
    if (e >= 0) row = of_warp[warp * E + e] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) of_warp[warp * E + e] += __popc(same);
    __syncwarp();
    if (i < a.slots) {
      const bool fits = row >= 0 && row < a.rows;
      a.slot[i] = fits ? row : -1;
      if (fits) {
        a.position[row] = (int32_t)i;
        a.token[row] = (int32_t)((uint32_t)i / (uint32_t)a.k);
      }
    }
  }
  // padding: the ends of the runs, a warp each, and what lies behind the last
  for (int e = blockIdx.x * warps + warp; e < E; e += a.parts * warps) {
    const int64_t end = (int64_t)start[e] + plan_run(count[e], a.align);
    for (int64_t r = (int64_t)start[e] + count[e] + lane; r < end && r < a.rows; r += 32) {
      a.position[r] = -1;
      a.token[r] = -1;
    }
  }
  const int64_t used = (int64_t)start[E - 1] + plan_run(count[E - 1], a.align);
  for (int64_t r = used + (int64_t)blockIdx.x * threads + tid; r < a.rows; r += (int64_t)a.parts * threads) {
    a.position[r] = -1;
    a.token[r] = -1;
  }
}

// Warps a CTA has (shared memory holds a word for each of them and an expert), slots a lane has, parts.
static void plan_split(int64_t slots, int32_t experts, int* warps, int* each, int64_t* parts) {
  *warps = experts <= 512 ? 16 : 8;
  const int64_t lanes = (int64_t)*warps * 32;
  // up to 128 parts before a lane gets more than one slot (262 144 slots over 256 experts: 12.8 us of placing, 13.3 in 64)
  int64_t e = ceil_div(slots, lanes * PLAN_DIRECT);
  *each = (int)(e < 1 ? 1 : e > PLAN_EACH ? PLAN_EACH : e);
  if (slots <= lanes * PLAN_EACH) *each = (int)(slots <= lanes ? 1 : ceil_div(slots, lanes));   // one part, one launch
  *parts = slots <= 0 ? 1 : ceil_div(slots, lanes * *each);
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
  const bool bf16 = p->dtype == ALTOB200_DT_BF16;
  a.computed = bias != nullptr || a.group_top > 1;
  a.checked = a.computed || !bf16;
  a.score_room = !a.computed ? 0.0f : a.sigmoid ? 1.3e-6f : 1.5e-5f;
  a.per = (E + 31) / 32;
  const int size = E / a.groups, lanes = size % a.per == 0 ? size / a.per : 0;
  a.lanes_per_group = lanes > 0 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
  // a lane's logits as vectors: as many as the kernel has room for, in rows aligned to them
  const int bytes = a.per * (bf16 ? 2 : 4), width = bytes < 16 ? bytes : 16;
  const bool whole = E % 32 == 0 && (a.per & (a.per - 1)) == 0 && (reinterpret_cast<uintptr_t>(logits) % width) == 0 &&
                     (ld * (bf16 ? 2 : 4)) % width == 0;
  a.scratch = a.checked || a.groups > 1 ? (E > 64 ? E : 64) : 0;   // keys in double, or E words and 32 between groups
  const size_t smem = (size_t)8 * a.scratch * 8;
  int64_t blocks = ceil_div(tokens, 8);
  if (blocks > 148 * 4) blocks = 148 * 4;
  if (blocks < ceil_div(tokens, 8 * 32)) blocks = ceil_div(tokens, 8 * 32);
  if (blocks >= (1ll << 31)) return ALTOB200_ELIMIT;
#define RUN(B, V)                                                                                                           \
  (void)launch_after(whole ? route_forward_kernel<B, V, true> : route_forward_kernel<B, V, false>, dim3((unsigned)blocks), \
                     dim3(256), smem, (cudaStream_t)stream, a)
  if (bf16) ROUTE_BY_V(RUN, true);
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
  a.vector = (reinterpret_cast<uintptr_t>(grad_logits) & 15) == 0 && (p->experts * (p->dtype == ALTOB200_DT_BF16 ? 2 : 4)) % 16 == 0;
  const int E = p->experts;
  if (a.sigmoid || a.renorm) {
    int64_t blocks = ceil_div(tokens, 16);
    if (blocks > 148 * 16) blocks = 148 * 16;
    (void)launch_after(p->dtype == ALTOB200_DT_BF16 ? route_backward_chosen_kernel<true> : route_backward_chosen_kernel<false>,
                       dim3((unsigned)blocks), dim3(256), 0, (cudaStream_t)stream, a);
    return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
  }
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
  int warps, each;
  int64_t parts;
  plan_split(slots, experts, &warps, &each, &parts);
  return parts > 1 ? (parts + 1) * experts * 4 : 0;
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
  int warps;
  int64_t parts;
  plan_split(slots, experts, &warps, &a.each, &parts);
  a.parts = (int32_t)parts;
  if (a.parts > 1 && work == nullptr) return ALTOB200_EINVAL_SHAPE;
  const cudaStream_t st = (cudaStream_t)stream;
  if (a.parts > 1) (void)launch_after(plan_count_kernel, dim3(a.parts), dim3(warps * 32), (size_t)experts * 4, st, a);
  if (a.parts > PLAN_DIRECT) (void)launch_after(plan_sum_kernel, dim3((experts + 31) / 32), dim3(1024), 0, st, a);
  (void)launch_after(plan_place_kernel, dim3(a.parts), dim3(warps * 32), (size_t)experts * (warps + 3) * 4, st, a);
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}
