// Root-mean-square norm of rows, with the residual's addition in front of it and with its result in the type of x or as
// MXFP8 codes and scales, and its backward pass.
//
//   r = T(x + residual)                     (r = x without one; T the type of x, because r is the stream that is stored)
//   y = T(r * rstd * w),  rstd = 1 / sqrt(mean(r^2) + eps)
//   dr = T(rstd * (dy w - xhat * mean(dy w xhat)) + d_stream),  dw = sum over rows of dy xhat,  xhat = r rstd
//
// Sums, rstd and dw are fp32; y is rounded once.  The 8-bit result is what altob200_quantize_rowwise makes of y (blocks
// of 32 along the row), so that both ways to the block-scaled product give the same codes.
//
// Both directions are HBM streams: forward reads x (and the residual) and writes y (and r), backward reads dy, r (and
// d_stream) and writes dr.  rstd is not kept: backward reads r anyway, and one more sum costs less than the launch-time
// allocation of a vector.  bf16 8192 x 4096 with residual (41 us a direction at the measured copy rate, a reference and no
// floor: streams that read more than they write run a little above it): forward 42 us, backward 43 and 4 to join dw;
// without loads ahead 68 and 5.  32768 x 4096 (164): 157 and 161 + 4.
//
// A row is held in registers: 16-byte vectors of it per thread (lane-adjacent, so that four (bf16) or eight (fp32)
// neighbouring lanes hold a block of 32) or, where width, strides or pointers rule those out, single elements.  8 to 32
// lanes of a warp hold a narrow row, a CTA a wide one; rows beyond 1024 threads x 4 vectors (16 elements forward, 8
// backward) take the kernels that read a row a second time.
#include "common.cuh"

namespace altob200 {

struct NormArgs {
  const void* x;
  const void* res;      // NULL: none
  const void* w;
  void* y;              // T [rows, cols], or the codes
  void* r;              // T [rows, cols], only with res
  void* y2;             // with codes: y as T [rows, cols] besides, or NULL
  uint8_t* scale_plain; // [rows, cols / 32] or NULL
  uint8_t* scale_packed;
  int64_t rows, cols, ld_x, ld_res;
  float eps, inv_cols;
  int32_t w_f32, e5m2;
};

template <bool BF16>
struct NormType;
template <>
struct NormType<true> {
  using T = __nv_bfloat16;
  static constexpr int V = 8;
};
template <>
struct NormType<false> {
  using T = float;
  static constexpr int V = 4;
};

// the elements of a 16-byte vector
template <bool BF16>
__device__ __forceinline__ void unpack_vec(const uint4& w, float* v) {
  if constexpr (BF16) {
    v[0] = bf16lo_to_f32(w.x); v[1] = bf16hi_to_f32(w.x); v[2] = bf16lo_to_f32(w.y); v[3] = bf16hi_to_f32(w.y);
    v[4] = bf16lo_to_f32(w.z); v[5] = bf16hi_to_f32(w.z); v[6] = bf16lo_to_f32(w.w); v[7] = bf16hi_to_f32(w.w);
  } else {
    v[0] = u2f(w.x); v[1] = u2f(w.y); v[2] = u2f(w.z); v[3] = u2f(w.w);
  }
}
template <bool BF16>
__device__ __forceinline__ uint4 pack_vec(const float* v) {
  if constexpr (BF16) {
    return make_uint4(pack_bf16_rn(v[0], v[1]), pack_bf16_rn(v[2], v[3]), pack_bf16_rn(v[4], v[5]), pack_bf16_rn(v[6], v[7]));
  } else {
    return make_uint4(f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3]));
  }
}
// What a thread holds at a time: a 16-byte vector, or (V = 1) one element.
template <int V>
struct Held { using U = uint4; };
template <>
struct Held<1> { using U = float; };

template <bool BF16>
__device__ __forceinline__ float load_elem(const void* p, int64_t i) {
  if constexpr (BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  else return reinterpret_cast<const float*>(p)[i];
}
template <bool BF16>
__device__ __forceinline__ void store_elem(void* p, int64_t i, float v) {
  if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}
template <bool BF16>
__device__ __forceinline__ float round_elem(float v) {
  return BF16 ? u2f(f32_to_bf16_bits(v) << 16) : v;
}
__device__ __forceinline__ float weight_elem(const void* w, int64_t i, int f32) {
  return f32 ? __ldg(reinterpret_cast<const float*>(w) + i) : __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16*>(w) + i));
}

template <bool BF16, int V>
__device__ __forceinline__ typename Held<V>::U load_unit(const void* row, int u) {
  if constexpr (V == 1) return load_elem<BF16>(row, u);
  else return __ldg(reinterpret_cast<const uint4*>(row) + u);
}
template <bool BF16, int V>
__device__ __forceinline__ void store_unit(void* row, int u, typename Held<V>::U v) {
  if constexpr (V == 1) store_elem<BF16>(row, u, v);
  else reinterpret_cast<uint4*>(row)[u] = v;
}
template <bool BF16, int V>
__device__ __forceinline__ void unpack_unit(const typename Held<V>::U& w, float* v) {
  if constexpr (V == 1) v[0] = w;
  else unpack_vec<BF16>(w, v);
}
template <bool BF16, int V>
__device__ __forceinline__ typename Held<V>::U pack_unit(const float* v) {
  if constexpr (V == 1) return round_elem<BF16>(v[0]);
  else return pack_vec<BF16>(v);
}
template <int V>
__device__ __forceinline__ typename Held<V>::U no_unit() {
  if constexpr (V == 1) return 0.0f;
  else return make_uint4(0u, 0u, 0u, 0u);
}

// V weights from column c, which is a multiple of V
template <int V>
__device__ __forceinline__ void load_weights(const void* w, int64_t c, int f32, float* out) {
  if constexpr (V == 1) {
    out[0] = weight_elem(w, c, f32);
  } else if (f32) {
#pragma unroll
    for (int q = 0; q < V; q += 4) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(w) + c + q));
      unpack_vec<false>(a, out + q);
    }
  } else if constexpr (V == 8) {
    unpack_vec<true>(__ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(w) + c)), out);
  } else {
    const uint2 a = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(w) + c));
    out[0] = bf16lo_to_f32(a.x); out[1] = bf16hi_to_f32(a.x); out[2] = bf16lo_to_f32(a.y); out[3] = bf16hi_to_f32(a.y);
  }
}

// Sum over groups of LANES lanes (every lane gets its group's).
template <int LANES = 32>
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// Sum over the CTA (every thread gets it).  `part` holds 32 values; callers that come again alternate between two.
__device__ __forceinline__ float block_sum(float v, float* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  v = warp_sum(v);
  if (lane == 0) part[warp] = v;
  __syncthreads();
  return warp_sum(lane < warps ? part[lane] : 0.0f);
}

// Codes of V values of one block of 32 that neighbouring lanes hold (already in the type of x): amax over the lanes, scale,
// encode.  Returns the scale byte.
template <bool BF16, int V, bool E5M2>
__device__ __forceinline__ uint32_t encode_block(const typename Held<V>::U& unit, uint8_t* to, bool store) {
  uint32_t m;   // largest magnitude, as bits of the type
  if constexpr (V == 8) {
    const uint32_t keep = 0x7FFF7FFFu;
    const uint32_t two = __vmaxu2(__vmaxu2(unit.x & keep, unit.y & keep), __vmaxu2(unit.z & keep, unit.w & keep));
    m = max(two >> 16, two & 0xFFFFu);
  } else if constexpr (V == 4) {
    m = max(max(unit.x & 0x7FFFFFFFu, unit.y & 0x7FFFFFFFu), max(unit.z & 0x7FFFFFFFu, unit.w & 0x7FFFFFFFu));
  } else {
    m = BF16 ? (f2u(unit) & 0x7FFFFFFFu) >> 16 : f2u(unit) & 0x7FFFFFFFu;
  }
  if constexpr (V == 1) {
    m = __reduce_max_sync(0xFFFFFFFFu, m);
  } else {
#pragma unroll
    for (int o = 1; o < 32 / V; o <<= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  }
  const uint32_t e = e8m0_from_amax_bits<BF16>(m, E5M2 ? 2 : 3, E5M2 ? 15 : 8);
  float s[V < 2 ? 2 : V];
  s[1] = 0.0f;
  unpack_unit<BF16, V>(unit, s);
  // 1 / 2^(e - 127): the formats' largest exponents keep e at 247 or below, for any bits of m
  const float r = u2f((254u - e) << 23);
  if constexpr (V == 1) {
    s[0] *= r;
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 p = __fmul2_rn(make_float2(s[j], s[j + 1]), make_float2(r, r));
      s[j] = p.x;
      s[j + 1] = p.y;
    }
  }
  if constexpr (V == 1) {
    if (store) *to = (uint8_t)fp8x2_rtn_hw<E5M2>(s[0], 0.0f);
  } else {
    uint32_t code[V / 4];
#pragma unroll
    for (int j = 0; j < V; j += 4) code[j / 4] = fp8x2_rtn_hw<E5M2>(s[j], s[j + 1]) | (fp8x2_rtn_hw<E5M2>(s[j + 2], s[j + 3]) << 16);
    if (store) {
      if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(code[0], code[1]);
      else *reinterpret_cast<uint32_t*>(to) = code[0];
    }
  }
  return e;
}

// Scale bytes of the packed layout that belong to no block: rows up to a multiple of 128, columns up to one of 4.
__device__ __forceinline__ void zero_packed_padding(const NormArgs& a, int64_t row, int thread, int threads) {
  const int64_t nkb = a.cols >> 5, tiles = (nkb + 3) >> 2;
  const int64_t first = row < a.rows ? nkb : 0;
  for (int64_t c = first + thread; c < tiles * 4; c += threads) a.scale_packed[packed_scale_offset(row, c, tiles)] = 0;
}

// One row per LANES lanes of a warp, or (LANES = 0) ROWS rows per CTA; NV units of V elements a thread and row.  FMT: 0 for
// the type of x, 1 e4m3, 2 e5m2.
//
// One row a CTA is bound by the turnover of CTAs, so two share one (8192 x 4096: 42 us, with codes 41; one by one 47 and
// 49), and with codes by instructions (issue slots 72 %), so elements go in pairs, maxima are taken of the packed words and
// scales are multiplied (with one element to an instruction and quotients 43).  The bounds keep three CTAs of 512 threads
// or two of 1024 on an SM: at 45 registers codes took 56 us.  CTAs that walk over rows with the next one's loads ahead, as in
// the backward pass, are slower (47, with codes 52), and scale bytes put together to words no faster.
template <bool BF16, int FMT, int LANES, int NV, int V, int ROWS = 1>
__global__ void __launch_bounds__(LANES ? 128 : ROWS > 1 ? 512 : 1024, LANES || NV > 2 ? 1 : ROWS > 1 ? 3 : 2) norm_forward_kernel(NormArgs a) {
  using T = typename NormType<BF16>::T;
  using U = typename Held<V>::U;
  constexpr bool WARP = LANES != 0, MX = FMT != 0;
  __shared__ float part[ROWS][32];
  grid_dependency_wait();
  const int threads = WARP ? LANES : blockDim.x, t = WARP ? (threadIdx.x & (LANES - 1)) : threadIdx.x;
  const int64_t first = WARP ? ((int64_t)blockIdx.x * 128 + threadIdx.x) / LANES : (int64_t)blockIdx.x * ROWS;
  if (MX && a.scale_packed != nullptr) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (first + k < ((a.rows + 127) & ~127ll)) zero_packed_padding(a, first + k, t, threads);
  }
  if (!WARP && first >= a.rows) return;
  U raw[ROWS][NV], add[ROWS][NV];
  // threads behind the last row go along with nothing
  const auto units_of = [&](int k) { return first + k < a.rows ? (int)(a.cols / V) : 0; };
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    const T* x = reinterpret_cast<const T*>(a.x) + (first + k) * a.ld_x;
    const T* res = reinterpret_cast<const T*>(a.res) + (first + k) * a.ld_res;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + i * threads;
      const bool on = u < units_of(k);
      raw[k][i] = on ? load_unit<BF16, V>(x, u) : no_unit<V>();
      if (a.res != nullptr) add[k][i] = on ? load_unit<BF16, V>(res, u) : no_unit<V>();
    }
  }
  float ss[ROWS];
#pragma unroll
  for (int k = 0; k < ROWS; ++k) {
    ss[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float p[V];
      unpack_unit<BF16, V>(raw[k][i], p);
      if (a.res != nullptr) {
        const int u = t + i * threads;
        float q[V];
        unpack_unit<BF16, V>(add[k][i], q);
        if constexpr (V == 1) {
          p[0] = __fadd_rn(p[0], q[0]);
        } else {
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const float2 n = __fadd2_rn(make_float2(p[j], p[j + 1]), make_float2(q[j], q[j + 1]));
            p[j] = n.x;
            p[j + 1] = n.y;
          }
        }
        raw[k][i] = pack_unit<BF16, V>(p);
        if (u < units_of(k)) store_unit<BF16, V>(reinterpret_cast<T*>(a.r) + (first + k) * a.cols, u, raw[k][i]);
        unpack_unit<BF16, V>(raw[k][i], p);
      }
      if constexpr (V == 1) {
        ss[k] = __fmaf_rn(p[0], p[0], ss[k]);
      } else {
        float2 two = make_float2(ss[k], 0.0f);
#pragma unroll
        for (int j = 0; j < V; j += 2) two = __ffma2_rn(make_float2(p[j], p[j + 1]), make_float2(p[j], p[j + 1]), two);
        ss[k] = two.x + two.y;
      }
    }
    ss[k] = warp_sum<WARP ? LANES : 32>(ss[k]);
  }
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
      if (lane == 0) part[k][warp] = ss[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ROWS; ++k) ss[k] = warp_sum(lane < warps ? part[k][lane] : 0.0f);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int u = t + i * threads;
    float w[V] = {};
    if (u < (int)(a.cols / V)) load_weights<V>(a.w, (int64_t)u * V, a.w_f32, w);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int64_t row = first + k;
      const bool on = u < units_of(k);
      const float rstd = rsqrtf(__fmaf_rn(ss[k], a.inv_cols, a.eps));
      float p[V];
      unpack_unit<BF16, V>(raw[k][i], p);
      if constexpr (V == 1) {
        p[0] = p[0] * rstd * w[0];
      } else {
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const float2 n = __fmul2_rn(__fmul2_rn(make_float2(p[j], p[j + 1]), make_float2(rstd, rstd)), make_float2(w[j], w[j + 1]));
          p[j] = n.x;
          p[j + 1] = n.y;
        }
      }
      const U y = pack_unit<BF16, V>(p);
      if constexpr (MX) {
        if (a.y2 != nullptr && on) store_unit<BF16, V>(reinterpret_cast<T*>(a.y2) + row * a.cols, u, y);
        const uint32_t e = encode_block<BF16, V, FMT == 2>(y, reinterpret_cast<uint8_t*>(a.y) + row * a.cols + (int64_t)u * V, on);
        constexpr int HOLD = 32 / V;   // lanes that hold one block
        if (on && (u & (HOLD - 1)) == 0) {
          const int64_t nkb = a.cols >> 5, kb = u / HOLD;
          if (a.scale_plain != nullptr) a.scale_plain[row * nkb + kb] = (uint8_t)e;
          if (a.scale_packed != nullptr) a.scale_packed[packed_scale_offset(row, kb, (nkb + 3) >> 2)] = (uint8_t)e;
        }
      } else if (on) {
        store_unit<BF16, V>(reinterpret_cast<T*>(a.y) + row * a.cols, u, y);
      }
    }
  }
}

// Any width, stride and alignment: one row per CTA, elements one by one, the row read again for the result.
template <bool BF16, bool MX>
__global__ void __launch_bounds__(256) norm_forward_any_kernel(NormArgs a) {
  __shared__ float part[32];
  grid_dependency_wait();
  const int64_t row = blockIdx.x;
  if (MX && a.scale_packed != nullptr) zero_packed_padding(a, row, threadIdx.x, 256);
  if (row >= a.rows) return;
  const auto stream = [&](int64_t c) {
    const float v = load_elem<BF16>(a.x, row * a.ld_x + c);
    return a.res == nullptr ? v : round_elem<BF16>(__fadd_rn(v, load_elem<BF16>(a.res, row * a.ld_res + c)));
  };
  float ss = 0.0f;
  for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
    const float v = stream(c);
    if (a.res != nullptr) store_elem<BF16>(a.r, row * a.cols + c, v);
    ss = __fmaf_rn(v, v, ss);
  }
  ss = block_sum(ss, part);
  const float rstd = rsqrtf(__fmaf_rn(ss, a.inv_cols, a.eps));
  for (int64_t c = threadIdx.x; c < a.cols; c += 256) {   // MX: cols is a multiple of 32, so whole warps come here
    const float v = stream(c) * rstd * weight_elem(a.w, c, a.w_f32);
    if constexpr (MX) {
      const float p = round_elem<BF16>(v);
      if (a.y2 != nullptr) store_elem<BF16>(a.y2, row * a.cols + c, p);
      uint32_t m = f2u(p) & 0x7FFFFFFFu;
      m = __reduce_max_sync(0xFFFFFFFFu, m);
      const uint32_t e = BF16 ? e8m0_from_amax_bits<true>(m >> 16, a.e5m2 ? 2 : 3, a.e5m2 ? 15 : 8)
                              : e8m0_from_amax_bits<false>(m, a.e5m2 ? 2 : 3, a.e5m2 ? 15 : 8);
      const float s = __fmul_rn(p, u2f((254u - e) << 23));
      reinterpret_cast<uint8_t*>(a.y)[row * a.cols + c] =
          (uint8_t)(a.e5m2 ? fp8x2_rtn_hw<true>(s, 0.0f) : fp8x2_rtn_hw<false>(s, 0.0f));
      if ((threadIdx.x & 31) == 0) {
        const int64_t nkb = a.cols >> 5, kb = c >> 5;
        if (a.scale_plain != nullptr) a.scale_plain[row * nkb + kb] = (uint8_t)e;
        if (a.scale_packed != nullptr) a.scale_packed[packed_scale_offset(row, kb, (nkb + 3) >> 2)] = (uint8_t)e;
      }
    } else {
      store_elem<BF16>(a.y, row * a.cols + c, v);
    }
  }
}

// ---------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------
struct NormGradArgs {
  const void* dy;
  const void* r;
  const void* ds;       // gradient of the stream, or NULL
  const void* w;
  void* dr;             // T [rows, cols]
  float* partial;       // [CTAs, cols], or NULL: no gradient of w
  int64_t rows, cols, ld_dy, ld_r, ld_ds;
  float eps, inv_cols;
  int32_t w_f32;
};

// Two sums over the CTA at once.
__device__ __forceinline__ float2 block_sum2(float u, float v, float2* part) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  u = warp_sum(u);
  v = warp_sum(v);
  if (lane == 0) part[warp] = make_float2(u, v);
  __syncthreads();
  const float2 p = lane < warps ? part[lane] : make_float2(0.0f, 0.0f);
  return make_float2(warp_sum(p.x), warp_sum(p.y));
}

// A CTA (or LANES lanes of it) walks over rows; a thread keeps its columns, so it sums their part of dw in registers and
// writes it once, a narrow row's groups of lanes through shared memory.  With one vector or four elements a thread
// (the usual widths; 64 registers hold no more) the next row's loads go out before the CTA meets over this row's sums, and
// the weights stay in registers.
template <bool BF16, int LANES, int NV, int V>
__global__ void __launch_bounds__(LANES ? 128 : 1024) norm_backward_kernel(NormGradArgs a) {
  using T = typename NormType<BF16>::T;
  using U = typename Held<V>::U;
  constexpr bool WARP = LANES != 0, AHEAD = V == 1 ? NV <= 4 : NV == 1;
  constexpr int GROUPS = WARP ? 128 / (WARP ? LANES : 1) : 1;
  __shared__ float2 part[2][32];
  extern __shared__ float joined[];   // WARP: [cols], the groups' sums
  grid_dependency_wait();
  const int threads = WARP ? LANES : blockDim.x, t = WARP ? (threadIdx.x & (LANES - 1)) : threadIdx.x;
  const int group = WARP ? threadIdx.x / (WARP ? LANES : 1) : 0;
  const int units = (int)(a.cols / V);
  float acc[NV][V] = {};
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  U g_next[NV], x_next[NV], d_next[NV];
  const auto load = [&](int64_t from) {
    const T* dy = reinterpret_cast<const T*>(a.dy) + from * a.ld_dy;
    const T* r = reinterpret_cast<const T*>(a.r) + from * a.ld_r;
    const T* ds = reinterpret_cast<const T*>(a.ds) + from * a.ld_ds;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + i * threads;
      const bool on = u < units && (!WARP || from < a.rows);
      g_next[i] = on ? load_unit<BF16, V>(dy, u) : no_unit<V>();
      x_next[i] = on ? load_unit<BF16, V>(r, u) : no_unit<V>();
      d_next[i] = on && a.ds != nullptr ? load_unit<BF16, V>(ds, u) : no_unit<V>();
    }
  };
  float w_kept[AHEAD ? NV : 1][V];
  if (AHEAD)
#pragma unroll
    for (int i = 0; i < (AHEAD ? NV : 1); ++i)
      if (t + i * threads < units) load_weights<V>(a.w, (int64_t)(t + i * threads) * V, a.w_f32, w_kept[i]);
  const auto weights = [&](int i, int u, float* w) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int j = 0; j < V; ++j) w[j] = w_kept[i][j];
    } else {
      load_weights<V>(a.w, (int64_t)u * V, a.w_f32, w);
    }
  };
  if (AHEAD && (WARP || row < a.rows)) load(row);
  // the groups of a warp stay together: all go on while the first has a row
  const int64_t first = row - (WARP ? (threadIdx.x & 31) / (WARP ? LANES : 1) : 0);
  for (int64_t lead = first; lead < a.rows; lead += step, row += step) {
    U g[NV], x[NV], ds[NV];
    if (!AHEAD) load(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      g[i] = g_next[i];
      x[i] = x_next[i];
      ds[i] = d_next[i];
    }
    if (AHEAD && (WARP || row + step < a.rows)) load(row + step);
    float ss = 0.0f, dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + i * threads;
      float gv[V], xv[V], w[V] = {};
      unpack_unit<BF16, V>(g[i], gv);
      unpack_unit<BF16, V>(x[i], xv);
      if (u < units) weights(i, u, w);
      if constexpr (V == 1 || NV > 1) {   // pairs cost registers that more units do not leave
#pragma unroll
        for (int j = 0; j < V; ++j) {
          ss = __fmaf_rn(xv[j], xv[j], ss);
          dot = __fmaf_rn(gv[j] * w[j], xv[j], dot);
        }
      } else {
        float2 s2 = make_float2(ss, 0.0f), d2 = make_float2(dot, 0.0f);
#pragma unroll
        for (int j = 0; j < V; j += 2) {
          const float2 xx = make_float2(xv[j], xv[j + 1]);
          s2 = __ffma2_rn(xx, xx, s2);
          d2 = __ffma2_rn(__fmul2_rn(make_float2(gv[j], gv[j + 1]), make_float2(w[j], w[j + 1])), xx, d2);
        }
        ss = s2.x + s2.y;
        dot = d2.x + d2.y;
      }
    }
    if constexpr (WARP) {
      ss = warp_sum<LANES>(ss);
      dot = warp_sum<LANES>(dot);
    } else {
      const float2 s = block_sum2(ss, dot, part[turn]);
      turn ^= 1;
      ss = s.x;
      dot = s.y;
    }
    const float rstd = rsqrtf(__fmaf_rn(ss, a.inv_cols, a.eps));
    const float along = dot * rstd * rstd * a.inv_cols;   // mean(dy w xhat) rstd
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + i * threads;
      if (u < units && (!WARP || row < a.rows)) {
        float gv[V], xv[V], w[V], d[V];
        unpack_unit<BF16, V>(g[i], gv);
        unpack_unit<BF16, V>(x[i], xv);
        unpack_unit<BF16, V>(ds[i], d);
        weights(i, u, w);
        if constexpr (V == 1 || NV > 1) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            acc[i][j] = __fmaf_rn(gv[j], xv[j] * rstd, acc[i][j]);
            d[j] = __fmaf_rn(rstd, __fmaf_rn(-xv[j], along, gv[j] * w[j]), d[j]);
          }
        } else {
          const float2 rr = make_float2(rstd, rstd), back = make_float2(-along, -along);
#pragma unroll
          for (int j = 0; j < V; j += 2) {
            const float2 gg = make_float2(gv[j], gv[j + 1]), xx = make_float2(xv[j], xv[j + 1]);
            const float2 sum = __ffma2_rn(gg, __fmul2_rn(xx, rr), make_float2(acc[i][j], acc[i][j + 1]));
            acc[i][j] = sum.x;
            acc[i][j + 1] = sum.y;
            const float2 gw = __fmul2_rn(gg, make_float2(w[j], w[j + 1]));
            const float2 to = __ffma2_rn(rr, __ffma2_rn(xx, back, gw), make_float2(d[j], d[j + 1]));
            d[j] = to.x;
            d[j + 1] = to.y;
          }
        }
        store_unit<BF16, V>(reinterpret_cast<T*>(a.dr) + row * a.cols, u, pack_unit<BF16, V>(d));
      }
    }
  }
  if (a.partial == nullptr) return;
  float* out = a.partial + (int64_t)blockIdx.x * a.cols;
  if constexpr (WARP) {
    for (int c = threadIdx.x; c < (int)a.cols; c += 128) joined[c] = 0.0f;
    for (int k = 0; k < GROUPS; ++k) {   // one after the other: the order of the sum is fixed
      __syncthreads();
      if (group == k) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int u = t + i * threads;
          if (u < units)
#pragma unroll
            for (int j = 0; j < V; ++j) joined[u * V + j] += acc[i][j];
        }
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < (int)a.cols; c += 128) out[c] = joined[c];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int u = t + i * threads;
      if (u < units) {
        if constexpr (V == 1) {
          out[u] = acc[i][0];
        } else {
#pragma unroll
          for (int j = 0; j < V; j += 4)
            *reinterpret_cast<float4*>(out + (int64_t)u * V + j) = make_float4(acc[i][j], acc[i][j + 1], acc[i][j + 2], acc[i][j + 3]);
        }
      }
    }
  }
}

// Any width, stride and alignment: the gradient of the rows, and behind it dw with a thread per column.
template <bool BF16>
__global__ void __launch_bounds__(256) norm_backward_any_kernel(NormGradArgs a) {
  __shared__ float2 part[2][32];
  grid_dependency_wait();
  int turn = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float ss = 0.0f, dot = 0.0f;
    for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
      const float g = load_elem<BF16>(a.dy, row * a.ld_dy + c), x = load_elem<BF16>(a.r, row * a.ld_r + c);
      ss = __fmaf_rn(x, x, ss);
      dot = __fmaf_rn(g * weight_elem(a.w, c, a.w_f32), x, dot);
    }
    const float2 s = block_sum2(ss, dot, part[turn]);
    turn ^= 1;
    const float rstd = rsqrtf(__fmaf_rn(s.x, a.inv_cols, a.eps)), along = s.y * rstd * rstd * a.inv_cols;
    float* out = a.partial == nullptr ? nullptr : a.partial + (int64_t)blockIdx.x * a.cols;
    for (int64_t c = threadIdx.x; c < a.cols; c += 256) {
      const float g = load_elem<BF16>(a.dy, row * a.ld_dy + c), x = load_elem<BF16>(a.r, row * a.ld_r + c);
      const float d = a.ds == nullptr ? 0.0f : load_elem<BF16>(a.ds, row * a.ld_ds + c);
      store_elem<BF16>(a.dr, row * a.cols + c, __fmaf_rn(rstd, __fmaf_rn(-x, along, g * weight_elem(a.w, c, a.w_f32)), d));
      // the thread's own columns: no other thread writes them
      if (out != nullptr) out[c] = (row == (int64_t)blockIdx.x ? 0.0f : out[c]) + g * (x * rstd);
    }
  }
}

// dw[c] = sum of the CTAs' parts, in a fixed order: 32 columns a CTA, its 32 warps over the parts.
__global__ void __launch_bounds__(1024) norm_join_kernel(const float* __restrict__ partial, int parts, int64_t cols,
                                                         void* __restrict__ dw, int w_f32) {
  __shared__ float sums[32][33];
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < cols) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 32) s += __ldg(partial + p * cols + c);
  }
  sums[warp][lane] = s;
  __syncthreads();
  // warp w: column w of the 32
  s = warp_sum(sums[lane][warp]);
  const int64_t of = (int64_t)blockIdx.x * 32 + warp;
  if (lane == 0 && of < cols) {
    if (w_f32) reinterpret_cast<float*>(dw)[of] = s;
    else reinterpret_cast<__nv_bfloat16*>(dw)[of] = __float2bfloat16_rn(s);
  }
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a row is spread.  lanes: of a warp, 0: a CTA of `threads`; nv: units a thread; v: elements a unit (1 or a 16-byte
// vector); threads = 0: the kernels for any width.
struct NormShape {
  int lanes, threads, nv, v;
};
static NormShape norm_shape(int64_t cols, int vec, bool forward) {
  if (vec > 1) {
    const int64_t units = cols / vec;
    if (units <= 32) return {units <= 8 ? 8 : units <= 16 ? 16 : 32, 128, 1, vec};
    // forward: two vectors a thread rather than CTAs of more than 512 (4096 x 8192 bf16 with codes 55 us in two rows a CTA)
    const int nv = units <= (forward ? 512 : 1024) ? 1 : units <= 2048 ? 2 : 4;
    if (units <= 4096) return {0, (int)(ceil_div(ceil_div(units, nv), 32) * 32), nv, vec};
    return {0, 0, 0, 0};
  }
  // four elements a thread keep a backward pass's loads ahead; forward is faster with eight (11650 x 2879: fp32 102 us
  // against 113, bf16 113 against 125)
  if (cols <= 128) return {32, 128, 4, 1};
  const int nv = !forward && cols <= 4096 ? 4 : cols <= 8192 ? 8 : 16;
  if (cols <= 8192 || (forward && cols <= 16384)) return {0, (int)(ceil_div(ceil_div(cols, nv), 32) * 32), nv, 1};
  return {0, 0, 0, 0};
}

// CTAs of a backward pass, no more than there are rows for.  A CTA a row: what the SMs hold at 64 registers a thread.  A few
// lanes a row: eight a SM, of which five to seven fit at a time (72 to 95 registers), so that the last run in a second,
// emptier round: 262144 x 128 bf16 54 us where the bytes take 41.
static int norm_blocks_backward(const NormShape& s, int64_t rows) {
  if (s.threads == 0) return (int)(rows < 148 * 4 ? rows : 148 * 4);
  const int64_t all = s.lanes ? ceil_div(rows, 128 / s.lanes) : rows;
  const int64_t most = 148 * (s.lanes ? 8 : 1024 / s.threads);
  return (int)(all < most ? all : most);
}

}  // namespace altob200

using namespace altob200;

extern "C" int altob200_rms_norm_forward(const altob200_rms_norm_args* p, void* stream) {
  if (p == nullptr || p->rows < 0 || p->cols <= 0) return ALTOB200_EINVAL_SHAPE;
  if (p->rows == 0) return ALTOB200_OK;
  const bool bf16 = p->dtype == ALTOB200_DT_BF16, mx = p->format >= 0;
  if ((!bf16 && p->dtype != ALTOB200_DT_F32) || (p->weight_dtype != ALTOB200_DT_BF16 && p->weight_dtype != ALTOB200_DT_F32) ||
      (mx && p->format != ALTOB200_FMT_MXFP8_E4M3 && p->format != ALTOB200_FMT_MXFP8_E5M2))
    return ALTOB200_EUNSUPPORTED;
  if (p->x == nullptr || p->weight == nullptr || p->out == nullptr || p->ld_x < p->cols ||
      (p->residual != nullptr && (p->stream_out == nullptr || p->ld_residual < p->cols)) ||
      (!mx && p->normed_out != nullptr) || (mx && (p->cols % 32 != 0 || (p->scale_plain == nullptr && p->scale_packed == nullptr))))
    return ALTOB200_EINVAL_SHAPE;
  if (p->rows >= (1ll << 31) - 128) return ALTOB200_ELIMIT;
  const int V = bf16 ? 8 : 4;
  const bool vec = p->cols % V == 0 && p->ld_x % V == 0 && aligned16(p->x) && aligned16(p->out) && aligned16(p->weight) && aligned16(p->normed_out) &&
                   (p->residual == nullptr || (p->ld_residual % V == 0 && aligned16(p->residual) && aligned16(p->stream_out)));
  const NormShape s = norm_shape(p->cols, vec ? V : 1, true);
  NormArgs a;
  a.x = p->x; a.res = p->residual; a.w = p->weight; a.y = p->out; a.r = p->stream_out; a.y2 = p->normed_out;
  a.scale_plain = p->scale_plain; a.scale_packed = p->scale_packed;
  a.rows = p->rows; a.cols = p->cols; a.ld_x = p->ld_x; a.ld_res = p->ld_residual;
  a.eps = p->eps; a.inv_cols = (float)(1.0 / (double)p->cols);
  a.w_f32 = p->weight_dtype == ALTOB200_DT_F32;
  a.e5m2 = p->format == ALTOB200_FMT_MXFP8_E5M2;
  const int64_t all_rows = mx && p->scale_packed != nullptr ? ceil_div(p->rows, 128) * 128 : p->rows;
  const cudaStream_t st = (cudaStream_t)stream;
  if (s.threads == 0) {
#define ANY(B, M) (void)launch_after(norm_forward_any_kernel<B, M>, dim3((unsigned)all_rows), dim3(256), 0, st, a)
    if (bf16) { if (mx) ANY(true, true); else ANY(true, false); }
    else { if (mx) ANY(false, true); else ANY(false, false); }
#undef ANY
  } else {
    // two rows a CTA as soon as there are more rows than CTAs at a time (4096 columns: 148 rows 2.1 us one by one, 2.4 in
    // pairs; 2400 rows 10.3 and 9.4, 8192 rows 47 and 42, with codes 49 and 41)
    const bool two = s.lanes == 0 && s.nv == 1 && s.v > 1 && all_rows > 148 * 4;
    const dim3 grid((unsigned)(s.lanes ? ceil_div(all_rows, 128 / s.lanes) : two ? ceil_div(all_rows, 2) : all_rows)), block(s.threads);
#define ONE(B, M, L, N, V) (void)launch_after(norm_forward_kernel<B, M, L, N, V>, grid, block, 0, st, a)
#define BY_SHAPE(B, M, V)                             \
  do {                                                \
    if (s.v == 1) {                                   \
      if (s.lanes) ONE(B, M, 32, 4, 1);               \
      else if (s.nv == 8) ONE(B, M, 0, 8, 1);         \
      else ONE(B, M, 0, 16, 1);                       \
    } else if (s.lanes == 8) ONE(B, M, 8, 1, V);      \
    else if (s.lanes == 16) ONE(B, M, 16, 1, V);      \
    else if (s.lanes == 32) ONE(B, M, 32, 1, V);      \
    else if (two) (void)launch_after(norm_forward_kernel<B, M, 0, 1, V, 2>, grid, block, 0, st, a); \
    else if (s.nv == 1) ONE(B, M, 0, 1, V);           \
    else if (s.nv == 2) ONE(B, M, 0, 2, V);           \
    else ONE(B, M, 0, 4, V);                          \
  } while (0)
    if (bf16) { if (!mx) BY_SHAPE(true, 0, 8); else if (!a.e5m2) BY_SHAPE(true, 1, 8); else BY_SHAPE(true, 2, 8); }
    else { if (!mx) BY_SHAPE(false, 0, 4); else if (!a.e5m2) BY_SHAPE(false, 1, 4); else BY_SHAPE(false, 2, 4); }
#undef BY_SHAPE
#undef ONE
  }
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

static bool norm_backward_vec(const altob200_rms_norm_grad_args* p) {
  const int V = p->dtype == ALTOB200_DT_BF16 ? 8 : 4;
  return p->cols % V == 0 && p->ld_grad % V == 0 && p->ld_stream % V == 0 && aligned16(p->grad_out) && aligned16(p->stream) &&
         aligned16(p->weight) && aligned16(p->grad_in) &&
         (p->grad_stream == nullptr || (p->ld_grad_stream % V == 0 && aligned16(p->grad_stream)));
}

extern "C" int64_t altob200_rms_norm_backward_work_bytes(const altob200_rms_norm_grad_args* p) {
  if (p == nullptr || p->rows <= 0 || p->cols <= 0 || p->grad_weight == nullptr) return 0;
  const NormShape s = norm_shape(p->cols, norm_backward_vec(p) ? (p->dtype == ALTOB200_DT_BF16 ? 8 : 4) : 1, false);
  return (int64_t)norm_blocks_backward(s, p->rows) * p->cols * 4;
}

extern "C" int altob200_rms_norm_backward(const altob200_rms_norm_grad_args* p, void* work, void* stream) {
  if (p == nullptr || p->rows < 0 || p->cols <= 0) return ALTOB200_EINVAL_SHAPE;
  const bool bf16 = p->dtype == ALTOB200_DT_BF16;
  if ((!bf16 && p->dtype != ALTOB200_DT_F32) || (p->weight_dtype != ALTOB200_DT_BF16 && p->weight_dtype != ALTOB200_DT_F32))
    return ALTOB200_EUNSUPPORTED;
  const cudaStream_t st = (cudaStream_t)stream;
  const int w_f32 = p->weight_dtype == ALTOB200_DT_F32;
  if (p->rows == 0) {   // a sum over no rows
    if (p->grad_weight != nullptr) ALTOB200_CUDA_CHECK(cudaMemsetAsync(p->grad_weight, 0, p->cols * (w_f32 ? 4 : 2), st));
    return ALTOB200_OK;
  }
  if (p->grad_out == nullptr || p->stream == nullptr || p->weight == nullptr || p->grad_in == nullptr || p->ld_grad < p->cols ||
      p->ld_stream < p->cols || (p->grad_stream != nullptr && p->ld_grad_stream < p->cols) ||
      (p->grad_weight != nullptr && work == nullptr))
    return ALTOB200_EINVAL_SHAPE;
  if (!aligned16(work)) return ALTOB200_EINVAL_ALIGN;
  if (p->rows >= (1ll << 31) - 128) return ALTOB200_ELIMIT;
  const NormShape s = norm_shape(p->cols, norm_backward_vec(p) ? (p->dtype == ALTOB200_DT_BF16 ? 8 : 4) : 1, false);
  const int blocks = norm_blocks_backward(s, p->rows);
  NormGradArgs a;
  a.dy = p->grad_out; a.r = p->stream; a.ds = p->grad_stream; a.w = p->weight; a.dr = p->grad_in;
  a.partial = p->grad_weight == nullptr ? nullptr : reinterpret_cast<float*>(work);
  a.rows = p->rows; a.cols = p->cols; a.ld_dy = p->ld_grad; a.ld_r = p->ld_stream; a.ld_ds = p->ld_grad_stream;
  a.eps = p->eps; a.inv_cols = (float)(1.0 / (double)p->cols); a.w_f32 = w_f32;
  if (s.threads == 0) {
    if (bf16) (void)launch_after(norm_backward_any_kernel<true>, dim3(blocks), dim3(256), 0, st, a);
    else (void)launch_after(norm_backward_any_kernel<false>, dim3(blocks), dim3(256), 0, st, a);
  } else {
    const size_t smem = s.lanes ? (size_t)p->cols * 4 : 0;
#define ONE(B, L, N, V) (void)launch_after(norm_backward_kernel<B, L, N, V>, dim3(blocks), dim3(s.threads), smem, st, a)
#define BY_SHAPE(B, V)                             \
  do {                                             \
    if (s.v == 1) {                                \
      if (s.lanes) ONE(B, 32, 4, 1);               \
      else if (s.nv == 4) ONE(B, 0, 4, 1);         \
      else ONE(B, 0, 8, 1);                        \
    } else if (s.lanes == 8) ONE(B, 8, 1, V);      \
    else if (s.lanes == 16) ONE(B, 16, 1, V);      \
    else if (s.lanes == 32) ONE(B, 32, 1, V);      \
    else if (s.nv == 1) ONE(B, 0, 1, V);           \
    else if (s.nv == 2) ONE(B, 0, 2, V);           \
    else ONE(B, 0, 4, V);                          \
  } while (0)
    if (bf16) BY_SHAPE(true, 8);
    else BY_SHAPE(false, 4);
#undef BY_SHAPE
#undef ONE
  }
  if (p->grad_weight != nullptr)
    (void)launch_after(norm_join_kernel, dim3((unsigned)ceil_div(p->cols, 32)), dim3(1024), 0, st, (const float*)a.partial,
                       blocks, p->cols, p->grad_weight, w_f32);
  return cudaGetLastError() == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}
