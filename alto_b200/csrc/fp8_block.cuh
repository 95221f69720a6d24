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

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <bool E5M2>
__device__ __forceinline__ float fp8b_scale(float amax) {
  return __fdiv_rn(max_nan(amax, FP8B_LEAST), E5M2 ? 57344.0f : 448.0f);
}
// What the quotients by a scale take: (s, RN(1 / s)).  The reciprocal forms of common.cuh hold for every scale there is, 2^-56 to
// 2^120: a quotient that any code but zero stands for keeps its residual normal, and one below that may be off.  Behind an
// infinite scale every number but the infinities and NaN has quotient zero, which (0, 0) gives.
__device__ __forceinline__ float2 fp8b_divisor(float s) {
  return s == __int_as_float(0x7F800000) ? make_float2(0.0f, 0.0f) : make_float2(s, __frcp_rn(s));
}
// x / s of two numbers in packed arithmetic (the roundings of div_bf16_num and div_f32_num)
template <bool BF16>
__device__ __forceinline__ float2 fp8b_quotients(float a, float b, float2 f) {
  const float2 x = make_float2(a, b), s2 = make_float2(f.x, f.x), n2 = make_float2(-f.y, -f.y), m2 = make_float2(-a, -b);
  float2 y = __fmul2_rn(x, make_float2(f.y, f.y));
  if (!BF16) y = __ffma2_rn(n2, __ffma2_rn(y, s2, m2), y);
  return __ffma2_rn(n2, __ffma2_rn(y, s2, m2), y);
}
// The codes of four numbers of one block as a word.
template <bool BF16, bool E5M2>
__device__ __forceinline__ uint32_t fp8b_word(float a, float b, float c, float d, float2 f) {
  const float2 p = fp8b_quotients<BF16>(a, b, f), q = fp8b_quotients<BF16>(c, d, f);
  uint32_t w;
  if (E5M2)
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e5m2x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e5m2x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(w) : "f"(p.x), "f"(p.y), "f"(q.x), "f"(q.y));
  else
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
        "mov.b32 %0, {lo, hi};\n\t}"
        : "=r"(w) : "f"(p.x), "f"(p.y), "f"(q.x), "f"(q.y));
  return w;
}

// Rows of expert e: ends are device memory that no host has seen, so they are taken as they would be in order and inside
// the buffer (a running maximum, cut off at the buffer's rows).
struct Fp8bRun {
  int expert;      // -1: none
  int row0, row1;  // rows of the run
  int unit;        // of the run
};
// The run that holds unit `at` where every run is cut into units of `size` rows, by one warp.
__device__ __forceinline__ Fp8bRun fp8b_find(const int32_t* offs, int experts, int64_t rows, int at, int size) {
  Fp8bRun r = {-1, 0, 0, 0};
  const int lane = threadIdx.x & 31;
  int carry_end = 0, carry_units = 0;
  for (int e0 = 0; e0 < experts; e0 += 32) {
    const int e = e0 + lane;
    int end = e < experts ? __ldg(offs + e) : 0;
    end = end < 0 ? 0 : (int64_t)end > rows ? (int)rows : end;
    int start = __shfl_up_sync(0xFFFFFFFFu, end, 1);
    if (lane == 0) start = carry_end;
    if (!__all_sync(0xFFFFFFFFu, end >= start || e >= experts)) {      // not in order
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xFFFFFFFFu, end, d);
        if (lane >= d && o > end) end = o;
      }
      if (end < carry_end) end = carry_end;
      start = __shfl_up_sync(0xFFFFFFFFu, end, 1);
      if (lane == 0) start = carry_end;
    }
    if (e >= experts) end = start = 0;
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
      r.unit = at - __shfl_sync(0xFFFFFFFFu, before, src);
      return r;
    }
    carry_end = __shfl_sync(0xFFFFFFFFu, end, 31);      // (of no use behind the last experts)
    carry_units = __shfl_sync(0xFFFFFFFFu, before + n, 31);
  }
  return r;
}

}  // namespace altob200
