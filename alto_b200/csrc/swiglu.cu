// SwiGLU between the two grouped GEMMs of an expert MLP, forward and backward, one kernel each.
//
//   forward   out[r, c]      = bf16( bf16(silu(g)) * u ),   g = h[r, c], u = h[r, H + c]
//   backward  grad_h[r, c]   = bf16( bf16(go * u) * s * (1 + g * (1 - s)) ),   s = 1 / (1 + exp(-g))
//             grad_h[r, H+c] = bf16( go * bf16(silu(g)) )
//
// The expert MLP that the reference converts (the GroupedExperts module of its TorchTitan fork,
// alto/modifiers/lpt/base.py:186-187; the module itself is not among the reference's sources) puts a
// SiLU-gated product between its grouped GEMMs.  With the gate and up projections fused into one
// GEMM that writes [rows, 2H], tensor ops on the two halves cost eight passes over the routed rows
// forward and backward.  Intermediate roundings to bf16 are kept where the tensor-op form
// silu(h[:, :H]) * h[:, H:] and its autograd have them, so that the values equal that form's.
//
// One thread handles 8 columns of one row (16-byte loads and stores); both kernels are plain HBM
// streams: forward reads 4H and writes 2H bytes per row, backward reads 6H and writes 4H.
#include "common.cuh"

namespace altob200 {

__device__ __forceinline__ float silu_f32(float g) { return g / (1.0f + expf(-g)); }

__device__ __forceinline__ void unpack8(const uint4& w, float v[8]) {
  v[0] = bf16lo_to_f32(w.x); v[1] = bf16hi_to_f32(w.x); v[2] = bf16lo_to_f32(w.y); v[3] = bf16hi_to_f32(w.y);
  v[4] = bf16lo_to_f32(w.z); v[5] = bf16hi_to_f32(w.z); v[6] = bf16lo_to_f32(w.w); v[7] = bf16hi_to_f32(w.w);
}
__device__ __forceinline__ uint4 pack8(const float v[8]) {
  uint4 o;
  o.x = f32_to_bf16_bits(v[0]) | (f32_to_bf16_bits(v[1]) << 16);
  o.y = f32_to_bf16_bits(v[2]) | (f32_to_bf16_bits(v[3]) << 16);
  o.z = f32_to_bf16_bits(v[4]) | (f32_to_bf16_bits(v[5]) << 16);
  o.w = f32_to_bf16_bits(v[6]) | (f32_to_bf16_bits(v[7]) << 16);
  return o;
}
__device__ __forceinline__ float round_bf16(float x) { return u2f(f32_to_bf16_bits(x) << 16); }

template <bool BACKWARD>
__global__ void __launch_bounds__(256) swiglu_kernel(const uint4* __restrict__ h, const uint4* __restrict__ go,
                                                     int64_t rows, int64_t hv /* H / 8 */, int64_t ldv /* ld_h / 8 */,
                                                     uint4* __restrict__ out) {
  grid_dependency_wait();
  const int64_t n = rows * hv;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / hv, c = i - r * hv;
    float g[8], u[8];
    unpack8(__ldg(h + r * ldv + c), g);
    unpack8(__ldg(h + r * ldv + hv + c), u);
    if (!BACKWARD) {
      float o[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = __fmul_rn(round_bf16(silu_f32(g[j])), u[j]);
      out[r * hv + c] = pack8(o);
    } else {
      float d[8], dg[8], du[8];
      unpack8(__ldg(go + r * hv + c), d);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float s = 1.0f / (1.0f + expf(-g[j]));
        const float ds = round_bf16(__fmul_rn(d[j], u[j]));
        dg[j] = ds * s * (1.0f + g[j] * (1.0f - s));
        du[j] = __fmul_rn(d[j], round_bf16(silu_f32(g[j])));
      }
      out[r * ldv + c] = pack8(dg);
      out[r * ldv + hv + c] = pack8(du);
    }
  }
}

static int swiglu_launch(const void* h, const void* go, int64_t rows, int64_t H, int64_t ld_h, void* out, bool backward,
                         cudaStream_t st) {
  if (rows == 0) return ALTOB200_OK;
  if (h == nullptr || out == nullptr || (backward && go == nullptr) || rows < 0 || H <= 0 || ld_h < 2 * H)
    return ALTOB200_EINVAL_SHAPE;
  if (H % 8 != 0 || ld_h % 8 != 0 || (reinterpret_cast<uintptr_t>(h) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (backward && (reinterpret_cast<uintptr_t>(go) & 15)))
    return ALTOB200_EINVAL_ALIGN;
  int64_t blocks = ceil_div(rows * (H / 8), 256);
  if (blocks > 148 * 16) blocks = 148 * 16;
  if (backward)
    (void)launch_after(swiglu_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, st, reinterpret_cast<const uint4*>(h), reinterpret_cast<const uint4*>(go),
                                                          rows, H / 8, ld_h / 8, reinterpret_cast<uint4*>(out));
  else
    (void)launch_after(swiglu_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, st, reinterpret_cast<const uint4*>(h), nullptr, rows, H / 8, ld_h / 8,
                                                           reinterpret_cast<uint4*>(out));
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

// ---------------------------------------------------------------------------------------
// The same activation with its input kept for the backward pass as MXFP8 (codes and one E8M0 scale for 32 neighbours of
// a row, what altob200_quantize_rowwise makes of h) instead of bf16: 1.03 bytes an element for 2.
//
// Forward writes the result of swiglu_kernel, bit for bit, and the codes from the same read of h.  Backward decodes
// g and u and evaluates
//   grad_h[r, c] = bf16( go u s (1 + g (1 - s)) ),  grad_h[r, H + c] = bf16( go g s )
// in fp32 with one rounding: the tensor-op form's intermediate roundings are of an h that no longer exists here.
//
// 69632 x 2880 (floor 247 us a direction: 8.06 and 8.06 bytes a column at the copy rate): forward 272 us, bound by
// instructions; backward 252, the copy rate.  With expf and divisions 396 and 460; forward without the loads ahead 278, with
// one number to an instruction 282 (290 instructions for eight columns of both halves, issue slots 74 % busy).
// ---------------------------------------------------------------------------------------
// 16 / (1 + e^-g), off by the steps of the exponential and of the reciprocal.  The factor 16 keeps the reciprocal of
// 1 + e^88.7 above the least normal number; a sixteenth of a bf16 number is exact.  Outside of +-126, where the result is 16
// or 0, g is cut; a NaN comes back with the product that every caller forms with g.
__device__ __forceinline__ float sigmoid16(float g) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fmaf_rn(fast_exp(-fminf(fmaxf(g, -126.0f), 126.0f)), 0.0625f, 0.0625f)));
  return r;
}
// Two at once, for the direction that has no more instructions to spare (in the other their pairs of registers cost more
// warps than they save: 258 us for 252).
__device__ __forceinline__ float2 sigmoid16(float2 g) {
  const float2 e = fast_exp2x(make_float2(-fminf(fmaxf(g.x, -126.0f), 126.0f), -fminf(fmaxf(g.y, -126.0f), 126.0f)));
  const float2 d = __ffma2_rn(e, make_float2(0.0625f, 0.0625f), make_float2(0.0625f, 0.0625f));
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  return r;
}
__device__ __forceinline__ uint4 pack8_rn(const float v[8]) {
  return make_uint4(pack_bf16_rn(v[0], v[1]), pack_bf16_rn(v[2], v[3]), pack_bf16_rn(v[4], v[5]), pack_bf16_rn(v[6], v[7]));
}

// Scale byte of a block from the largest magnitude (bf16 bits), and eight of its elements (two to a word) as codes.
template <bool E5M2>
__device__ __forceinline__ uint2 encode8_mxfp8(const float v[8], uint32_t e) {
  float s[8];
  // 1 / 2^(e - 127): the formats' largest exponents keep e at 247 or below, for any bits of the maximum
  const float r = u2f((254u - e) << 23);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 p = __fmul2_rn(make_float2(v[j], v[j + 1]), make_float2(r, r));
    s[j] = p.x;
    s[j + 1] = p.y;
  }
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) w[j] = fp8x2_rtn_hw<E5M2>(s[4 * j], s[4 * j + 1]) | (fp8x2_rtn_hw<E5M2>(s[4 * j + 2], s[4 * j + 3]) << 16);
  return make_uint2(w[0], w[1]);
}
// Largest magnitude (as bits) of the two halves' eight elements.
__device__ __forceinline__ uint32_t absmax8_bits(const uint4& w) {
  const uint32_t m = 0x7FFF7FFFu;
  const uint32_t a = __vmaxu2(__vmaxu2(w.x & m, w.y & m), __vmaxu2(w.z & m, w.w & m));
  return max(a >> 16, a & 0xFFFFu);
}

// Where a thread is in [rows, hv] when it walks with the grid: one division at the start, none in the loop.
struct SwigluWalk {
  int64_t r, dr;
  int c, dc;
  __device__ __forceinline__ SwigluWalk(int hv) {
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
    r = i / hv;
    c = (int)(i - r * hv);
    dr = step / hv;
    dc = (int)(step - dr * hv);
  }
  __device__ __forceinline__ void next(int hv) {
    r += dr;
    c += dc;
    if (c >= hv) {
      c -= hv;
      ++r;
    }
  }
};

// Eight columns of gate and up a thread; four neighbouring lanes, which run together because hv is a multiple of four, hold
// a block of gate and one of up, whose maxima share the words of two shuffles.
template <bool E5M2>
__global__ void __launch_bounds__(256) swiglu_keep_kernel(const uint4* __restrict__ h, int64_t rows, int hv, int64_t ldv,
                                                          uint4* __restrict__ out, uint2* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  grid_dependency_wait();
  const unsigned lanes = 0xFu << (threadIdx.x & 28);
  SwigluWalk at(hv), ahead = at;
  uint4 wg_next = {}, wu_next = {};
  if (at.r < rows) {
    wg_next = __ldg(h + at.r * ldv + at.c);
    wu_next = __ldg(h + at.r * ldv + hv + at.c);
  }
  for (; at.r < rows; at = ahead) {
    const uint4 wg = wg_next, wu = wu_next;
    ahead.next(hv);
    if (ahead.r < rows) {   // the next vectors are on their way while these are worked on
      wg_next = __ldg(h + ahead.r * ldv + ahead.c);
      wu_next = __ldg(h + ahead.r * ldv + hv + ahead.c);
    }
    float g[8], u[8], o[8];
    unpack8(wg, g);
    unpack8(wu, u);
    uint32_t m = absmax8_bits(wg) | (absmax8_bits(wu) << 16);
    m = __vmaxu2(m, __shfl_xor_sync(lanes, m, 1));
    m = __vmaxu2(m, __shfl_xor_sync(lanes, m, 2));
    const uint32_t eg = e8m0_from_amax_bits<true>(m & 0xFFFFu, E5M2 ? 2 : 3, E5M2 ? 15 : 8);
    const uint32_t eu = e8m0_from_amax_bits<true>(m >> 16, E5M2 ? 2 : 3, E5M2 ? 15 : 8);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const float2 two = make_float2(g[j], g[j + 1]);
      const float2 silu = __fmul2_rn(__fmul2_rn(two, make_float2(0.0625f, 0.0625f)), sigmoid16(two));
      const uint32_t w = pack_bf16_rn(silu.x, silu.y);
      const float2 p = __fmul2_rn(make_float2(bf16lo_to_f32(w), bf16hi_to_f32(w)), make_float2(u[j], u[j + 1]));
      o[j] = p.x;
      o[j + 1] = p.y;
    }
    out[at.r * hv + at.c] = pack8_rn(o);
    codes[at.r * 2 * hv + at.c] = encode8_mxfp8<E5M2>(g, eg);
    codes[at.r * 2 * hv + hv + at.c] = encode8_mxfp8<E5M2>(u, eu);
    if ((threadIdx.x & 3) == 0) {
      const int nb = hv >> 2, b = at.c >> 2;
      scales[at.r * 2 * nb + b] = (uint8_t)eg;
      scales[at.r * 2 * nb + nb + b] = (uint8_t)eu;
    }
  }
}

template <bool E5M2>
__device__ __forceinline__ void decode8_mxfp8(const uint2& w, uint32_t e, float v[8]) {
  const float q = u2f(e << 23);   // the quantizers' scales are 2^-126 at least
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t two = ((j < 2 ? w.x : w.y) >> (16 * (j & 1))) & 0xFFFFu;
    const float2 f = __fmul2_rn(fp8x2_decode<E5M2>(two), make_float2(q, q));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

template <bool E5M2>
__global__ void __launch_bounds__(256) swiglu_kept_backward_kernel(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                   const uint4* __restrict__ go, int64_t rows, int hv,
                                                                   uint4* __restrict__ out) {
  grid_dependency_wait();
  const int nb = hv >> 2;
  for (SwigluWalk at(hv); at.r < rows; at.next(hv)) {
    const uint2 wg = __ldg(codes + at.r * 2 * hv + at.c), wu = __ldg(codes + at.r * 2 * hv + hv + at.c);
    const uint32_t eg = __ldg(scales + at.r * 2 * nb + (at.c >> 2)), eu = __ldg(scales + at.r * 2 * nb + nb + (at.c >> 2));
    const uint4 wd = __ldg(go + at.r * hv + at.c);
    float g[8], u[8], d[8];
    unpack8(wd, d);
    decode8_mxfp8<E5M2>(wg, eg, g);
    decode8_mxfp8<E5M2>(wu, eu, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float s = __fmul_rn(sigmoid16(g[j]), 0.0625f), gs = __fmul_rn(g[j], s), ds = __fmul_rn(d[j], u[j]);
      g[j] = __fmul_rn(ds, __fmaf_rn(gs, __fsub_rn(1.0f, s), s));   // go u (s + g s (1 - s))
      u[j] = __fmul_rn(d[j], gs);
    }
    out[at.r * 2 * hv + at.c] = pack8_rn(g);
    out[at.r * 2 * hv + hv + at.c] = pack8_rn(u);
  }
}

// Backward gains from more and shorter walks (69632 x 2880: 284 us with 16 a SM, 252
// with 64), forward, whose walks start with loads that nothing covers, does not.
static unsigned swiglu_blocks(int64_t rows, int64_t H, int per_sm) {
  const int64_t blocks = ceil_div(rows * (H / 8), 256);
  return (unsigned)(blocks > 148 * per_sm ? 148 * per_sm : blocks);
}

}  // namespace altob200

extern "C" {

int altob200_swiglu_forward(const void* h, int64_t rows, int64_t H, int64_t ld_h, void* out, void* stream) {
  return altob200::swiglu_launch(h, nullptr, rows, H, ld_h, out, false, (cudaStream_t)stream);
}

int altob200_swiglu_backward(const void* h, const void* grad_out, int64_t rows, int64_t H, int64_t ld_h, void* grad_h,
                             void* stream) {
  return altob200::swiglu_launch(h, grad_out, rows, H, ld_h, grad_h, true, (cudaStream_t)stream);
}

int altob200_swiglu_keep_forward(const void* h, int64_t rows, int64_t H, int64_t ld_h, int32_t format, void* out, void* codes,
                                 uint8_t* scales, void* stream) {
  using namespace altob200;
  if (format != ALTOB200_FMT_MXFP8_E4M3 && format != ALTOB200_FMT_MXFP8_E5M2) return ALTOB200_EUNSUPPORTED;
  if (rows == 0) return ALTOB200_OK;
  if (H >= (1ll << 31)) return ALTOB200_ELIMIT;
  if (h == nullptr || out == nullptr || codes == nullptr || scales == nullptr || rows < 0 || H <= 0 || H % 32 != 0 || ld_h < 2 * H)
    return ALTOB200_EINVAL_SHAPE;
  if (ld_h % 8 != 0 || (reinterpret_cast<uintptr_t>(h) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (reinterpret_cast<uintptr_t>(codes) & 15))
    return ALTOB200_EINVAL_ALIGN;
  (void)launch_after(format == ALTOB200_FMT_MXFP8_E5M2 ? swiglu_keep_kernel<true> : swiglu_keep_kernel<false>, dim3(swiglu_blocks(rows, H, 16)), dim3(256), 0, (cudaStream_t)stream,
                     reinterpret_cast<const uint4*>(h), rows, (int)(H / 8), ld_h / 8,
                     reinterpret_cast<uint4*>(out), reinterpret_cast<uint2*>(codes), scales);
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

int altob200_swiglu_kept_backward(const void* codes, const uint8_t* scales, const void* grad_out, int64_t rows, int64_t H,
                                  int32_t format, void* grad_h, void* stream) {
  using namespace altob200;
  if (format != ALTOB200_FMT_MXFP8_E4M3 && format != ALTOB200_FMT_MXFP8_E5M2) return ALTOB200_EUNSUPPORTED;
  if (rows == 0) return ALTOB200_OK;
  if (H >= (1ll << 31)) return ALTOB200_ELIMIT;
  if (codes == nullptr || scales == nullptr || grad_out == nullptr || grad_h == nullptr || rows < 0 || H <= 0 || H % 32 != 0)
    return ALTOB200_EINVAL_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(grad_out) & 15) ||
      (reinterpret_cast<uintptr_t>(grad_h) & 15))
    return ALTOB200_EINVAL_ALIGN;
  (void)launch_after(format == ALTOB200_FMT_MXFP8_E5M2 ? swiglu_kept_backward_kernel<true> : swiglu_kept_backward_kernel<false>, dim3(swiglu_blocks(rows, H, 64)), dim3(256), 0, (cudaStream_t)stream,
                     reinterpret_cast<const uint2*>(codes), scales, reinterpret_cast<const uint4*>(grad_out), rows, (int)(H / 8),
                     reinterpret_cast<uint4*>(grad_h));
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

}  // extern "C"
