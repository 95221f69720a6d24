// Norm of many tensors together, and the tensors scaled to a largest norm.
//
//   norm = sqrt(sum of squares) or max |g|,   factor = min(1, max_norm / (norm + 1e-6)),   out = g * factor
//
// Bound by HBM: one read for the norm, one read and one write for the scaled ones (none where nothing is clipped and the
// tensors are scaled in place).  The tensors' addresses travel as kernel arguments, so a list costs no copy to the device
// and can be captured; the second pass walks from the end, which L2 still holds.  Pieces of 32 KB of one tensor are dealt out to
// eight blocks an SM.  1.74 GB in 36 bf16 tensors: norm 266 us (6.5 TB/s), scaling 580 (6.0); 2000 tensors of bf16 and fp32, 120 MB:
// two launches of 16 and 22 us and two of 16 and 28, where the host's walk over the pairs takes 130 to 145.
// Squares are summed in fp32 over 32 numbers of a thread and in fp64 from there on; where those 32 leave the range in which
// fp32 squares are exact to a step (below 2^-80, above 2^100, or not finite) they are summed again in fp64.  Every block leaves
// one partial sum and they are joined in order: the result does not depend on timing.
#include <type_traits>

#include "common.cuh"

namespace altob200 {

// Tensors of a launch.  Short lists travel in a short table: arguments of 28 KB take the host some microseconds.
constexpr int GN_TENSORS = 1000, GN_FEW = 128;
constexpr int GN_THREADS = 256;
constexpr int GN_UNROLL = 4;
constexpr int64_t GN_CHUNK = 8 * GN_THREADS;    // 16-byte vectors of a block's piece

template <int MOST>
struct GradTable {
  static constexpr int SIZE = MOST;
  const void* g[MOST];
  void* out[MOST];
  int64_t n[MOST];                          // elements * 2 + (1: fp32)
  uint32_t first[MOST + 1];                 // pieces of the tensors in front
  int count;
};
static_assert(sizeof(GradTable<GN_TENSORS>) <= 30000, "kernel arguments");

template <int MOST>
__device__ __forceinline__ int table_find(const GradTable<MOST>& t, uint32_t piece) {
  int lo = 0, hi = t.count - 1;             // the last tensor that begins at or before the piece (empty ones have none)
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= piece) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// A tensor's elements in front of its first 16-byte boundary.
__device__ __host__ __forceinline__ int64_t head_of(const void* p, int esz, int64_t n) {
  const int64_t h = (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / esz;
  return h < n ? h : n;
}

template <bool F32>
__device__ __forceinline__ float element(const void* p, int64_t i) {
  if (F32) return static_cast<const float*>(p)[i];
  return u2f((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
template <bool F32>
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[F32 ? 4 : 8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = (&v.x)[j];
    if (F32) {
      x[j] = u2f(w);
    } else {
      x[2 * j] = bf16lo_to_f32(w);
      x[2 * j + 1] = bf16hi_to_f32(w);
    }
  }
}

template <bool INF>
struct Sum {
  double total = 0.0;
  float most = 0.0f;
  template <bool F32, int N>
  __device__ __forceinline__ void add(const uint4 (&v)[N]) {
    if (INF) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float x[F32 ? 4 : 8];
        unpack<F32>(v[k], x);
#pragma unroll
        for (int j = 0; j < (F32 ? 4 : 8); j += 2) most = absmax3_nan(most, x[j], x[j + 1]);
      }
    } else {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float x[F32 ? 4 : 8];
        unpack<F32>(v[k], x);
#pragma unroll
        for (int j = 0; j < (F32 ? 4 : 8); ++j) s = __fmaf_rn(x[j], x[j], s);
      }
      if (s > 8.271806125530277e-25f && s < 1.2676506002282294e30f) {
        total += (double)s;
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) {
          if (((v[k].x | v[k].y | v[k].z | v[k].w) & (F32 ? 0x7FFFFFFFu : 0x7FFF7FFFu)) == 0u) continue;
          float x[F32 ? 4 : 8];
          unpack<F32>(v[k], x);
#pragma unroll
          for (int j = 0; j < (F32 ? 4 : 8); ++j) total += (double)x[j] * (double)x[j];
        }
      }
    }
  }
  __device__ __forceinline__ void one(float x) {
    if (INF) most = absmax3_nan(most, x, 0.0f);
    else total += (double)x * (double)x;
  }
};

__device__ __forceinline__ double join(double a, double b, bool inf) {
  if (!inf) return a + b;
  return a != a ? a : b != b ? b : a > b ? a : b;      // a NaN stays one
}
// Over the block, the same in every thread.
__device__ __forceinline__ double block_join(double v, bool inf, double* shared) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = join(v, __shfl_xor_sync(0xFFFFFFFFu, v, d), inf);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = shared[0];
  for (int w = 1; w < GN_THREADS / 32; ++w) r = join(r, shared[w], inf);
  return r;
}

template <bool F32, bool INF>
__device__ __forceinline__ void piece_sum(const void* p, int64_t n, int64_t piece, Sum<INF>& s) {
  constexpr int PER = F32 ? 4 : 8;
  const int64_t head = head_of(p, F32 ? 4 : 2, n), vectors = (n - head) / PER;
  const uint4* const v = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + head * (F32 ? 4 : 2));
  const int64_t end = (piece + 1) * GN_CHUNK < vectors ? (piece + 1) * GN_CHUNK : vectors;
  int64_t i = piece * GN_CHUNK + threadIdx.x;
  for (; i + (GN_UNROLL - 1) * GN_THREADS < end; i += GN_UNROLL * GN_THREADS) {
    uint4 x[GN_UNROLL];
#pragma unroll
    for (int u = 0; u < GN_UNROLL; ++u) x[u] = __ldg(v + i + u * GN_THREADS);
    s.template add<F32>(x);
  }
  for (; i < end; i += GN_THREADS) {
    const uint4 x[1] = {__ldg(v + i)};
    s.template add<F32>(x);
  }
  if (piece == 0) {      // what is in front of the vectors and behind them
    if ((int64_t)threadIdx.x < head) s.one(element<F32>(p, threadIdx.x));
    const int64_t at = head + vectors * PER + threadIdx.x;
    if (at < n) s.one(element<F32>(p, at));
  }
}

template <bool INF, int MOST>
__global__ void __launch_bounds__(GN_THREADS) grad_norm_kernel(const __grid_constant__ GradTable<MOST> t, double* parts) {
  __shared__ double shared[GN_THREADS / 32];
  grid_dependency_wait();
  Sum<INF> s;
  const uint32_t pieces = t.first[t.count];
  for (uint32_t p = blockIdx.x; p < pieces; p += gridDim.x) {
    const int i = table_find(t, p);
    const int64_t n = t.n[i] >> 1;
    if (t.n[i] & 1) piece_sum<true, INF>(t.g[i], n, p - t.first[i], s);
    else piece_sum<false, INF>(t.g[i], n, p - t.first[i], s);
  }
  const double r = block_join(INF ? (double)s.most : s.total, INF, shared);
  if (threadIdx.x == 0) parts[blockIdx.x] = r;
}

// Sum (or maximum) of the parts, the same in every thread of every block.
__device__ __forceinline__ double all_parts(const double* parts, int n, bool inf, double* shared) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += GN_THREADS) v = join(v, parts[i], inf);
  return block_join(v, inf, shared);
}

__global__ void __launch_bounds__(GN_THREADS) grad_norm_finish_kernel(const double* parts, int n, int inf, double* total, float* norm) {
  __shared__ double shared[GN_THREADS / 32];
  grid_dependency_wait();
  const double v = all_parts(parts, n, inf != 0, shared);
  if (threadIdx.x == 0) {
    if (total != nullptr) *total = v;
    if (norm != nullptr) *norm = (float)(inf ? v : sqrt(v));
  }
}

template <bool F32>
__device__ __forceinline__ uint4 scaled(const uint4& v, float f) {
  float x[F32 ? 4 : 8];
  unpack<F32>(v, x);
#pragma unroll
  for (int j = 0; j < (F32 ? 4 : 8); ++j) x[j] = __fmul_rn(x[j], f);
  if constexpr (F32) return make_uint4(f2u(x[0]), f2u(x[1]), f2u(x[2]), f2u(x[3]));
  else return make_uint4(pack_bf16_rn(x[0], x[1]), pack_bf16_rn(x[2], x[3]), pack_bf16_rn(x[4], x[5]), pack_bf16_rn(x[6], x[7]));
}
template <bool F32>
__device__ __forceinline__ void scale_one(const void* p, void* out, int64_t i, float f) {
  const float x = __fmul_rn(element<F32>(p, i), f);
  if (F32) static_cast<float*>(out)[i] = x;
  else static_cast<uint16_t*>(out)[i] = (uint16_t)f32_to_bf16_bits(x);
}

template <bool F32>
__device__ __forceinline__ void piece_scale(const void* p, void* out, int64_t n, int64_t piece, float f) {
  constexpr int PER = F32 ? 4 : 8;
  const int64_t head = head_of(p, F32 ? 4 : 2, n), vectors = (n - head) / PER;
  const uint4* const v = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + head * (F32 ? 4 : 2));
  char* const o = static_cast<char*>(out) + head * (F32 ? 4 : 2);
  const int64_t end = (piece + 1) * GN_CHUNK < vectors ? (piece + 1) * GN_CHUNK : vectors;
  if ((reinterpret_cast<uintptr_t>(o) & 15) == 0) {
    uint4* const w = reinterpret_cast<uint4*>(o);
    int64_t i = piece * GN_CHUNK + threadIdx.x;
    for (; i + (GN_UNROLL - 1) * GN_THREADS < end; i += GN_UNROLL * GN_THREADS) {
      uint4 x[GN_UNROLL];
#pragma unroll
      for (int u = 0; u < GN_UNROLL; ++u) x[u] = v[i + u * GN_THREADS];
#pragma unroll
      for (int u = 0; u < GN_UNROLL; ++u) w[i + u * GN_THREADS] = scaled<F32>(x[u], f);
    }
    for (; i < end; i += GN_THREADS) w[i] = scaled<F32>(v[i], f);
  } else {      // the two lie differently to 16 bytes
    const int64_t first = head + piece * GN_CHUNK * PER, last = head + end * PER;
    for (int64_t i = first + threadIdx.x; i < last; i += GN_THREADS) scale_one<F32>(p, out, i, f);
  }
  if (piece == 0) {
    if ((int64_t)threadIdx.x < head) scale_one<F32>(p, out, threadIdx.x, f);
    const int64_t at = head + vectors * PER + threadIdx.x;
    if (at < n) scale_one<F32>(p, out, at, f);
  }
}

template <int MOST>
__global__ void __launch_bounds__(GN_THREADS) grad_scale_kernel(const __grid_constant__ GradTable<MOST> t, const double* parts, int n_parts, int inf,
                                                                double max_norm, float* norm_out) {
  __shared__ double shared[GN_THREADS / 32];
  grid_dependency_wait();
  const double v = all_parts(parts, n_parts, inf != 0, shared), norm = inf ? v : sqrt(v);
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double q = max_norm / (norm + 1e-6);
  const float f = q > 1.0 ? 1.0f : (float)q;      // (a NaN stays one)
  const uint32_t pieces = t.first[t.count];
  for (uint32_t b = blockIdx.x; b < pieces; b += gridDim.x) {
    const uint32_t p = pieces - 1 - b;
    const int i = table_find(t, p);
    if (f == 1.0f && t.out[i] == t.g[i]) continue;
    const int64_t n = t.n[i] >> 1;
    if (t.n[i] & 1) piece_scale<true>(t.g[i], t.out[i], n, p - t.first[i], f);
    else piece_scale<false>(t.g[i], t.out[i], n, p - t.first[i], f);
  }
}

static int gn_sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  return n;
}
static int64_t pieces_of(const void* g, int64_t n, bool f32) {
  if (n == 0) return 0;
  const int64_t vectors = (n - head_of(g, f32 ? 4 : 2, n)) / (f32 ? 4 : 8);
  const int64_t p = ceil_div(vectors, GN_CHUNK);
  return p < 1 ? 1 : p;
}
constexpr int GN_BLOCKS_PER_SM = 8;

// Walks the list a launch at a time.  fn(table, blocks, launch's first partial) -> status
template <int MOST, class F>
static int walk_launches(const altob200_grad_list* l, int blocks_most, F fn) {
  int64_t i = 0;
  int parts = 0;
  while (i < l->count) {
    GradTable<MOST> t;
    t.count = 0;
    int64_t pieces = 0;
    while (i < l->count && t.count < MOST) {
      const int64_t n = l->sizes[i];
      const bool f32 = l->dtypes[i] == ALTOB200_DT_F32;
      if (n > 0) {
        const int64_t p = pieces_of(l->grads[i], n, f32);
        if (pieces + p >= (1ll << 31)) return ALTOB200_ELIMIT;
        const int k = t.count++;
        t.g[k] = l->grads[i];
        t.out[k] = l->outs != nullptr ? l->outs[i] : const_cast<void*>(l->grads[i]);
        t.n[k] = n * 2 + (f32 ? 1 : 0);
        t.first[k] = (uint32_t)pieces;
        pieces += p;
      }
      ++i;
    }
    if (t.count == 0) break;
    t.first[t.count] = (uint32_t)pieces;
    const int blocks = (int)(pieces < blocks_most ? pieces : blocks_most);
    const int rc = fn(t, blocks, parts);
    if (rc != ALTOB200_OK) return rc;
    parts += blocks;
  }
  return ALTOB200_OK;
}

template <class F>
static int for_each_launch(const altob200_grad_list* l, int blocks_most, F fn) {
  return l->count <= GN_FEW ? walk_launches<GN_FEW>(l, blocks_most, fn) : walk_launches<GN_TENSORS>(l, blocks_most, fn);
}

static int check_list(const altob200_grad_list* l) {
  if (l == nullptr || l->count < 0 || (l->count > 0 && (l->grads == nullptr || l->sizes == nullptr || l->dtypes == nullptr))) return ALTOB200_EINVAL_SHAPE;
  for (int64_t i = 0; i < l->count; ++i) {
    if (l->sizes[i] < 0 || (l->sizes[i] > 0 && (l->grads[i] == nullptr || (l->outs != nullptr && l->outs[i] == nullptr)))) return ALTOB200_EINVAL_SHAPE;
    if (l->dtypes[i] != ALTOB200_DT_BF16 && l->dtypes[i] != ALTOB200_DT_F32) return ALTOB200_EUNSUPPORTED;
    const uintptr_t m = l->dtypes[i] == ALTOB200_DT_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(l->grads[i]) & m) || (l->outs != nullptr && (reinterpret_cast<uintptr_t>(l->outs[i]) & m))) return ALTOB200_EINVAL_ALIGN;
  }
  return ALTOB200_OK;
}

}  // namespace altob200

using namespace altob200;

extern "C" {

int64_t altob200_grad_norm_work_bytes(int64_t count) {
  return count <= 0 ? 8 : ceil_div(count, GN_TENSORS) * (int64_t)gn_sms() * GN_BLOCKS_PER_SM * 8;
}

static int launch_parts(const altob200_grad_list* l, int norm_inf, double* parts, int* n_parts, cudaStream_t st) {
  *n_parts = 0;
  return for_each_launch(l, gn_sms() * GN_BLOCKS_PER_SM, [&](const auto& t, int blocks, int first) {
    constexpr int MOST = std::decay_t<decltype(t)>::SIZE;
    const cudaError_t e = norm_inf ? launch_after(grad_norm_kernel<true, MOST>, dim3(blocks), dim3(GN_THREADS), 0, st, t, parts + first)
                                   : launch_after(grad_norm_kernel<false, MOST>, dim3(blocks), dim3(GN_THREADS), 0, st, t, parts + first);
    *n_parts = first + blocks;
    return e == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
  });
}

int altob200_grad_norm(const altob200_grad_list* list, int32_t norm_inf, void* work, double* total, float* norm, void* stream) {
  int rc = check_list(list);
  if (rc != ALTOB200_OK) return rc;
  if (work == nullptr || (reinterpret_cast<uintptr_t>(work) & 7)) return ALTOB200_EINVAL_ALIGN;
  int n = 0;
  rc = launch_parts(list, norm_inf, (double*)work, &n, (cudaStream_t)stream);
  if (rc != ALTOB200_OK) return rc;
  const cudaError_t e = launch_after(grad_norm_finish_kernel, dim3(1), dim3(GN_THREADS), 0, (cudaStream_t)stream, (const double*)work, n,
                                     (int)norm_inf, total, norm);
  return e == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

int altob200_clip_grads(const altob200_grad_list* list, int32_t norm_inf, double max_norm, const double* total, void* work, float* norm,
                        void* stream) {
  int rc = check_list(list);
  if (rc != ALTOB200_OK) return rc;
  const double* parts = total;
  int n = 1;
  cudaStream_t st = (cudaStream_t)stream;
  if (total == nullptr) {
    if (work == nullptr || (reinterpret_cast<uintptr_t>(work) & 7)) return ALTOB200_EINVAL_ALIGN;
    parts = (const double*)work;
    rc = launch_parts(list, norm_inf, (double*)work, &n, st);
    if (rc != ALTOB200_OK) return rc;
  }
  bool said = false;
  rc = for_each_launch(list, gn_sms() * GN_BLOCKS_PER_SM, [&](const auto& t, int blocks, int) {
    constexpr int MOST = std::decay_t<decltype(t)>::SIZE;
    const cudaError_t e = launch_after(grad_scale_kernel<MOST>, dim3(blocks), dim3(GN_THREADS), 0, st, t, parts, n, (int)norm_inf, max_norm,
                                       said ? (float*)nullptr : norm);
    said = true;
    return e == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
  });
  if (rc != ALTOB200_OK || said || norm == nullptr) return rc;
  // no tensor has an element
  const cudaError_t e = launch_after(grad_norm_finish_kernel, dim3(1), dim3(GN_THREADS), 0, st, parts, total == nullptr ? 0 : 1, (int)norm_inf,
                                     (double*)nullptr, norm);
  return e == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

}  // extern "C"
