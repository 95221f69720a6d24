// FP8 with one fp32 scale for each block of 128: scale, quotient and codes, and the runs of ragged experts, as every kernel
// of this format computes them.
//
// A block's scale is s = max(|largest|, 1e-12) / top (top: 448 for E4M3, 57344 for E5M2), its codes are x / s rounded to the
// nearest, both quotients correctly rounded fp32.  An infinity or a NaN makes the scale one, and with it every product of
// the block.
#pragma once
#include "common.cuh"

namespace altob200 {

constexpr int FP8B = 128;      // numbers of a block
constexpr float FP8B_LEAST = 1e-12f;

template <bool E5M2>
__device__ __forceinline__ float fp8b_scale(float amax) {
  float a;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(a) : "f"(amax), "f"(FP8B_LEAST));
  return __fdiv_rn(a, E5M2 ? 57344.0f : 448.0f);
}
// x / s; r = RN(1 / s), fast: s within the range of the reciprocal forms (common.cuh)
template <bool BF16>
__device__ __forceinline__ float fp8b_quotient(float x, float s, float r, bool fast) {
  if (!fast) return __fdiv_rn(x, s);
  return BF16 ? div_bf16_num(x, s, r) : div_f32_num(x, s, r);
}

// Rows of expert e: ends are device memory that no host has seen, so they are taken as they would be in order and inside
// the buffer (a running maximum, cut off at the buffer's rows).
struct Fp8bRun {
  int expert;      // -1: none
  int row0, row1;  // rows of the run
  int unit;        // of the run
  int first;       // units of the runs in front
};
// The run that holds unit `at` where every run is cut into units of `size` rows, by one warp; rows behind the last run are a
// run of expert `experts` where `behind`.  offs == nullptr: one run of all rows.
__device__ __forceinline__ Fp8bRun fp8b_find(const int32_t* offs, int experts, int64_t rows, int at, int size, bool behind) {
  Fp8bRun r = {-1, 0, 0, 0, 0};
  if (offs == nullptr) {
    if ((int64_t)at * size < rows) r = {0, 0, (int)rows, at, 0};
    return r;
  }
  const int lane = threadIdx.x & 31, total = experts + (behind ? 1 : 0);
  int carry_end = 0, carry_units = 0;
  for (int e0 = 0; e0 < total; e0 += 32) {
    const int e = e0 + lane;
    int end = e < experts ? __ldg(offs + e) : (e == experts && behind) ? (int)rows : 0;
    end = end < 0 ? 0 : (int64_t)end > rows ? (int)rows : end;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, end, d);
      if (lane >= d && o > end) end = o;
    }
    if (end < carry_end) end = carry_end;
    int start = __shfl_up_sync(0xFFFFFFFFu, end, 1);
    if (lane == 0) start = carry_end;
    const int n = (end - start + size - 1) / size;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, sum, d);
      if (lane >= d) sum += o;
    }
    const int before = carry_units + sum - n;
    const uint32_t hit = __ballot_sync(0xFFFFFFFFu, at >= before && at < before + n);
    if (hit != 0) {
      const int src = __ffs((int)hit) - 1;
      r.expert = e0 + src;
      r.row0 = __shfl_sync(0xFFFFFFFFu, start, src);
      r.row1 = __shfl_sync(0xFFFFFFFFu, end, src);
      r.first = __shfl_sync(0xFFFFFFFFu, before, src);
      r.unit = at - r.first;
      return r;
    }
    carry_end = __shfl_sync(0xFFFFFFFFu, end, 31);
    carry_units = __shfl_sync(0xFFFFFFFFu, before + n, 31);
  }
  return r;
}

}  // namespace altob200
