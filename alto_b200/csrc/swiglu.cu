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
// ---------------------------------------------------------------------------------------
// Codes of eight elements; four neighbouring lanes hold a block of 32.  Returns the scale byte.
__device__ __forceinline__ uint32_t encode8_mxfp8(const float v[8], int e5m2, unsigned lanes, uint2* code) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, f2u(v[j]) & 0x7FFFFFFFu);
  m = max(m, __shfl_xor_sync(lanes, m, 1));
  m = max(m, __shfl_xor_sync(lanes, m, 2));
  const uint32_t e = e8m0_from_amax_bits<true>(m >> 16, e5m2 ? 2 : 3, e5m2 ? 15 : 8);
  const float q = u2f(e << 23), rq = u2f((254u - e) << 23);
  float s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[j] = e <= 253u ? __fmul_rn(v[j], rq) : __fdiv_rn(v[j], q);
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j)
    w[j] = e5m2 ? (fp8x2_rtn_hw<true>(s[4 * j], s[4 * j + 1]) | (fp8x2_rtn_hw<true>(s[4 * j + 2], s[4 * j + 3]) << 16))
                : (fp8x2_rtn_hw<false>(s[4 * j], s[4 * j + 1]) | (fp8x2_rtn_hw<false>(s[4 * j + 2], s[4 * j + 3]) << 16));
  *code = make_uint2(w[0], w[1]);
  return e;
}

// Eight columns of gate and up a thread.
__global__ void __launch_bounds__(256) swiglu_keep_kernel(const uint4* __restrict__ h, int64_t rows, int64_t hv, int64_t ldv,
                                                          int e5m2, uint4* __restrict__ out, uint2* __restrict__ codes,
                                                          uint8_t* __restrict__ scales) {
  grid_dependency_wait();
  const int64_t n = rows * hv;   // a multiple of 4, as hv is: four neighbouring lanes run together
  const unsigned lanes = 0xFu << (threadIdx.x & 28);
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / hv, c = i - r * hv;
    float g[8], u[8], o[8];
    unpack8(__ldg(h + r * ldv + c), g);
    unpack8(__ldg(h + r * ldv + hv + c), u);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = __fmul_rn(round_bf16(silu_f32(g[j])), u[j]);
    out[i] = pack8(o);
    uint2 kg, ku;
    const uint32_t eg = encode8_mxfp8(g, e5m2, lanes, &kg), eu = encode8_mxfp8(u, e5m2, lanes, &ku);
    codes[r * 2 * hv + c] = kg;
    codes[r * 2 * hv + hv + c] = ku;
    if ((threadIdx.x & 3) == 0) {
      const int64_t nb = hv >> 2, b = c >> 2;
      scales[r * 2 * nb + b] = (uint8_t)eg;
      scales[r * 2 * nb + nb + b] = (uint8_t)eu;
    }
  }
}

__device__ __forceinline__ void decode8_mxfp8(const uint2& w, uint32_t e, int e5m2, float v[8]) {
  const float q = e == 0u ? 5.877471754111438e-39f : u2f(e << 23);   // 2^(e - 127)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t two = ((j < 2 ? w.x : w.y) >> (16 * (j & 1))) & 0xFFFFu;
    const float2 f = e5m2 ? fp8x2_decode<true>(two) : fp8x2_decode<false>(two);
    v[2 * j] = f.x * q;
    v[2 * j + 1] = f.y * q;
  }
}

__global__ void __launch_bounds__(256) swiglu_kept_backward_kernel(const uint2* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                                   const uint4* __restrict__ go, int64_t rows, int64_t hv,
                                                                   int e5m2, uint4* __restrict__ out) {
  grid_dependency_wait();
  const int64_t n = rows * hv;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / hv, c = i - r * hv, nb = hv >> 2, b = c >> 2;
    float g[8], u[8], d[8], dg[8], du[8];
    decode8_mxfp8(__ldg(codes + r * 2 * hv + c), __ldg(scales + r * 2 * nb + b), e5m2, g);
    decode8_mxfp8(__ldg(codes + r * 2 * hv + hv + c), __ldg(scales + r * 2 * nb + nb + b), e5m2, u);
    unpack8(__ldg(go + i), d);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float s = 1.0f / (1.0f + expf(-g[j]));
      dg[j] = d[j] * u[j] * s * (1.0f + g[j] * (1.0f - s));
      du[j] = d[j] * g[j] * s;
    }
    out[r * 2 * hv + c] = pack8(dg);
    out[r * 2 * hv + hv + c] = pack8(du);
  }
}

static unsigned swiglu_blocks(int64_t rows, int64_t H) {
  const int64_t blocks = ceil_div(rows * (H / 8), 256);
  return (unsigned)(blocks > 148 * 16 ? 148 * 16 : blocks);
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
  if (h == nullptr || out == nullptr || codes == nullptr || scales == nullptr || rows < 0 || H <= 0 || H % 32 != 0 || ld_h < 2 * H)
    return ALTOB200_EINVAL_SHAPE;
  if (ld_h % 8 != 0 || (reinterpret_cast<uintptr_t>(h) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) ||
      (reinterpret_cast<uintptr_t>(codes) & 15))
    return ALTOB200_EINVAL_ALIGN;
  (void)launch_after(swiglu_keep_kernel, dim3(swiglu_blocks(rows, H)), dim3(256), 0, (cudaStream_t)stream,
                     reinterpret_cast<const uint4*>(h), rows, H / 8, ld_h / 8, (int)(format == ALTOB200_FMT_MXFP8_E5M2),
                     reinterpret_cast<uint4*>(out), reinterpret_cast<uint2*>(codes), scales);
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

int altob200_swiglu_kept_backward(const void* codes, const uint8_t* scales, const void* grad_out, int64_t rows, int64_t H,
                                  int32_t format, void* grad_h, void* stream) {
  using namespace altob200;
  if (format != ALTOB200_FMT_MXFP8_E4M3 && format != ALTOB200_FMT_MXFP8_E5M2) return ALTOB200_EUNSUPPORTED;
  if (rows == 0) return ALTOB200_OK;
  if (codes == nullptr || scales == nullptr || grad_out == nullptr || grad_h == nullptr || rows < 0 || H <= 0 || H % 32 != 0)
    return ALTOB200_EINVAL_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) & 15) || (reinterpret_cast<uintptr_t>(grad_out) & 15) ||
      (reinterpret_cast<uintptr_t>(grad_h) & 15))
    return ALTOB200_EINVAL_ALIGN;
  (void)launch_after(swiglu_kept_backward_kernel, dim3(swiglu_blocks(rows, H)), dim3(256), 0, (cudaStream_t)stream,
                     reinterpret_cast<const uint2*>(codes), scales, reinterpret_cast<const uint4*>(grad_out), rows, H / 8,
                     (int)(format == ALTOB200_FMT_MXFP8_E5M2), reinterpret_cast<uint4*>(grad_h));
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

}  // extern "C"
