// FP8 with one fp32 scale for each block of 128: quantizers and the products of few rows.
//
//   fp8b_quantize_kernel   rows (blocks of 128 columns), columns (blocks of 128 rows from every expert's first one, codes
//                          transposed) or both from one read; squares of 128 x 128 in either packing
//   fp8b_dequantize_kernel values of codes and scales
//   fp8b_rows_kernel       D = A B^T for up to eight rows of numbers, which it quantises itself, and for codes that no other
//                          kernel takes (lists of experts or places of scales past its limits, no columns to reduce)
// The products of few rows of codes are in gemm_fp8_stream.cuh, those of many in gemm_fp8_block.cuh.
#include "fp8_block.cuh"

namespace altob200 {

// ---------------------------------------------------------------------------------------
// quantizers
// ---------------------------------------------------------------------------------------
struct Fp8bQuant {
  const void* x;
  int64_t rows, cols, ld;
  const int32_t* offs;
  int experts;
  uint8_t* row_codes;    // [rows, cols]
  float* row_scales;     // [ceil(cols / 128), rows]
  uint8_t* col_codes;    // [cols, ld_col]
  int64_t ld_col;
  float* col_scales;     // [ld_col / 128, cols]
  int64_t x_batch;       // squares: elements between matrices
};
enum { FP8B_ROWS = 1, FP8B_COLS = 2, FP8B_SQUARES = 4 };

// Maxima of two non-negative bf16 a word, by their bits (a NaN is above an infinity).
__device__ __forceinline__ uint32_t max_halves(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// 8 x 8 numbers of a thread, and maxima of their magnitudes in a form that packs: two to a word from bf16, whose bits order
// them, or one fp32 a word.
template <class T>
struct Fp8bTile;
template <>
struct Fp8bTile<__nv_bfloat16> {
  static constexpr bool BF16 = true;
  static constexpr int WORDS = 4;      // of eight maxima
  uint4 v[8];
  __device__ __forceinline__ void load(int i, const void* base, int64_t at) { v[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + at)); }
  __device__ __forceinline__ void zero(int i) { v[i] = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ float get(int i, int j) const {
    const uint32_t w = (&v[i].x)[j >> 1];
    return (j & 1) ? bf16hi_to_f32(w) : bf16lo_to_f32(w);
  }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return max_halves(a, b); }
  // words of eight rows' maxima over this thread's columns, of eight columns' over its rows
  __device__ __forceinline__ void maxima(uint32_t (&rows)[4], uint32_t (&cols)[4], bool want_rows, bool want_cols) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) rows[j] = cols[j] = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t m = 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = (&v[i].x)[j] & 0x7FFF7FFFu;
        if (want_rows) m = max_halves(m, w);
        if (want_cols) cols[j] = max_halves(cols[j], w);
      }
      if (want_rows) {      // both halves in one, rows 2 k and 2 k + 1 a word
        m = max_halves(m, __byte_perm(m, 0, 0x1032));
        rows[i >> 1] = (i & 1) ? __byte_perm(rows[i >> 1], m, 0x5410) : m;
      }
    }
  }
  static __device__ __forceinline__ float value(uint32_t w, int half) { return half ? bf16hi_to_f32(w) : bf16lo_to_f32(w); }
  static __device__ __forceinline__ float whole(const uint32_t (&w)[4]) {
    const uint32_t m = max_halves(max_halves(w[0], w[1]), max_halves(w[2], w[3]));
    return max_nan(bf16lo_to_f32(m), bf16hi_to_f32(m));
  }
};
template <>
struct Fp8bTile<float> {
  static constexpr bool BF16 = false;
  static constexpr int WORDS = 8;
  float4 v[8][2];
  __device__ __forceinline__ void load(int i, const void* base, int64_t at) {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(base) + at);
    v[i][0] = __ldg(p);
    v[i][1] = __ldg(p + 1);
  }
  __device__ __forceinline__ void zero(int i) { v[i][0] = v[i][1] = make_float4(0, 0, 0, 0); }
  __device__ __forceinline__ float get(int i, int j) const { return (&v[i][j >> 2].x)[j & 3]; }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return a > b ? a : b; }      // magnitudes' bits
  __device__ __forceinline__ void maxima(uint32_t (&rows)[8], uint32_t (&cols)[8], bool want_rows, bool want_cols) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) rows[j] = cols[j] = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (want_rows) {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; j += 2) m = absmax3_nan(m, get(i, j), get(i, j + 1));
        rows[i] = f2u(m) & 0x7FFFFFFFu;
      }
    }
    if (want_cols)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) m = absmax3_nan(m, get(i, j), get(i + 1, j));
        cols[j] = f2u(m) & 0x7FFFFFFFu;
      }
  }
  static __device__ __forceinline__ float value(uint32_t w, int) { return u2f(w); }
  static __device__ __forceinline__ float whole(const uint32_t (&w)[8]) {
    float m = u2f(w[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) m = max_nan(m, u2f(w[i]));
    return m;
  }
};

// Four words whose bytes are four rows -> four words whose bytes are four columns.
__device__ __forceinline__ void transpose4(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
  const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
  a = __byte_perm(ab0, cd0, 0x5410);
  b = __byte_perm(ab0, cd0, 0x7632);
  c = __byte_perm(ab1, cd1, 0x5410);
  d = __byte_perm(ab1, cd1, 0x7632);
}

// Threads eight rows or columns apart read without conflicts.
__device__ __forceinline__ int fp8b_slot(int i) { return i + (i >> 3); }

// The codes of a thread's 8 x 8 numbers, along their rows and / or columns, and where they go.
template <class T, int WHAT, bool E5M2>
__device__ __forceinline__ void fp8b_emit(const Fp8bQuant& q, const Fp8bTile<T>& t, const float2* row_f, const float2* col_f, int row0, int row_end,
                                          int r_in, int c_in, int64_t col, int64_t chunk) {
  constexpr bool BF16 = Fp8bTile<T>::BF16;
  constexpr bool R = (WHAT & FP8B_ROWS) != 0, C = (WHAT & FP8B_COLS) != 0, S = (WHAT & FP8B_SQUARES) != 0;
  if (R || S) {
    uint2 words[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 f = row_f[S ? 0 : fp8b_slot(r_in + i)];
      words[i].x = fp8b_word<BF16, E5M2>(t.get(i, 0), t.get(i, 1), t.get(i, 2), t.get(i, 3), f);
      words[i].y = fp8b_word<BF16, E5M2>(t.get(i, 4), t.get(i, 5), t.get(i, 6), t.get(i, 7), f);
      const int64_t r = (int64_t)row0 + r_in + i;
      if (q.row_codes != nullptr && r < row_end)
        *reinterpret_cast<uint2*>(q.row_codes + ((S ? (int64_t)blockIdx.z * q.rows : 0) + r) * q.cols + col) = words[i];
    }
    if (S && q.col_codes != nullptr) {
      // (rows are a multiple of 16, so that a thread's eight are inside or outside together)
      if (row0 + r_in < row_end) {
        uint8_t* const out = q.col_codes + ((int64_t)blockIdx.z * q.cols + col) * q.ld_col + row0 + r_in;
        transpose4(words[0].x, words[1].x, words[2].x, words[3].x);
        transpose4(words[0].y, words[1].y, words[2].y, words[3].y);
        transpose4(words[4].x, words[5].x, words[6].x, words[7].x);
        transpose4(words[4].y, words[5].y, words[6].y, words[7].y);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint2*>(out + j * q.ld_col) =
              j < 4 ? make_uint2(words[j].x, words[j + 4].x) : make_uint2(words[j - 4].y, words[j].y);
      }
    }
  }
  if (C) {
    uint8_t* const out = q.col_codes + col * q.ld_col + chunk * 128 + r_in;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 f = col_f[fp8b_slot(c_in + j)];
      *reinterpret_cast<uint2*>(out + j * q.ld_col) =
          make_uint2(fp8b_word<BF16, E5M2>(t.get(0, j), t.get(1, j), t.get(2, j), t.get(3, j), f),
                     fp8b_word<BF16, E5M2>(t.get(4, j), t.get(5, j), t.get(6, j), t.get(7, j), f));
    }
  }
}

// A tile of 128 rows x 128 columns a CTA (256 threads), 8 x 8 numbers a thread, a warp 32 rows x 64 columns: a row's part of a
// warp is 128 bytes of bf16, a column's 32 bytes of codes.  8192 x 14336 bf16: both ways 102 us (4.6 TB/s), columns 63 (5.6), squares
// in both packings 78 (6.0).  Both ways is bound by instructions and their latency (17 an element, two quotients and their
// encoding among them; 24 warps an SM issue on 55 % of the cycles), the others come near HBM.  Runs of experts add a search
// of their ends a CTA, and tiles that are not full: 65536 x 5760 both ways 307 us without runs, 345 over 32 experts of as many rows each,
// 420 over 32 of 843 to 5791 rows, whose runs begin at any row.
template <class T, int WHAT, bool E5M2>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? (WHAT == (FP8B_ROWS | FP8B_COLS) ? 3 : 4) : 2) fp8b_quantize_kernel(const Fp8bQuant q) {
  constexpr bool R = (WHAT & FP8B_ROWS) != 0, C = (WHAT & FP8B_COLS) != 0, S = (WHAT & FP8B_SQUARES) != 0;
  __shared__ float row_max[2][128], col_max[4][128], whole[8];
  __shared__ float2 row_f[144], col_f[144];      // scale and its reciprocal, by fp8b_slot
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  int row0 = (int)blockIdx.y * 128, row_end = (int)q.rows;
  int64_t chunk = blockIdx.y;
  if (!S && q.offs != nullptr) {
    const Fp8bRun run = fp8b_find(q.offs, q.experts, q.rows, (int)blockIdx.y, 128);
    if (run.expert < 0) return;
    row0 = run.row0 + run.unit * 128;
    row_end = run.row1;
  }
  const int64_t col0 = (int64_t)blockIdx.x * 128;
  const int r_in = (warp & 3) * 32 + (lane >> 3) * 8, c_in = (warp >> 2) * 64 + (lane & 7) * 8;
  const int64_t col = col0 + c_in;
  const char* base = static_cast<const char*>(q.x) + (S ? (int64_t)blockIdx.z * q.x_batch * (int64_t)sizeof(T) : 0);
  Fp8bTile<T> t;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = (int64_t)row0 + r_in + i;
    if (r < row_end && col < q.cols) t.load(i, base, r * q.ld + col);
    else t.zero(i);
  }
  // largest magnitudes
  using Tile = Fp8bTile<T>;
  constexpr int W = Tile::WORDS;
  uint32_t rm[W], cm[W];
  t.maxima(rm, cm, R || S, C);
  if (S) {
    float m = Tile::whole(rm);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
    if (lane == 0) whole[warp] = m;
  }
  if (R) {
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) rm[i] = Tile::most(rm[i], __shfl_xor_sync(0xFFFFFFFFu, rm[i], d));
    if ((lane & 7) == 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) row_max[warp >> 2][r_in + i] = Tile::value(rm[i * W / 8], i & 1);
  }
  if (C) {
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int d = 8; d < 32; d <<= 1) cm[j] = Tile::most(cm[j], __shfl_xor_sync(0xFFFFFFFFu, cm[j], d));
    if (lane < 8)
#pragma unroll
      for (int j = 0; j < 8; ++j) col_max[warp & 3][c_in + j] = Tile::value(cm[j * W / 8], j & 1);
  }
  __syncthreads();
  // scales, a thread each
  if (S) {
    if (threadIdx.x == 0) {
      float m = whole[0];
      for (int w = 1; w < 8; ++w) m = max_nan(m, whole[w]);
      const float s = fp8b_scale<E5M2>(m);
      row_f[0] = fp8b_divisor(s);
      q.row_scales[((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s;
    }
  } else if (threadIdx.x < 128) {
    if (R) {
      const float s = fp8b_scale<E5M2>(max_nan(row_max[0][threadIdx.x], row_max[1][threadIdx.x]));
      row_f[fp8b_slot((int)threadIdx.x)] = fp8b_divisor(s);
      if (row0 + (int)threadIdx.x < row_end) q.row_scales[(int64_t)blockIdx.x * q.rows + row0 + threadIdx.x] = s;
    }
  } else if (C) {
    const int c = (int)threadIdx.x - 128;
    const float s = fp8b_scale<E5M2>(max_nan(max_nan(col_max[0][c], col_max[1][c]), max_nan(col_max[2][c], col_max[3][c])));
    col_f[fp8b_slot(c)] = fp8b_divisor(s);
    if (col0 + c < q.cols) q.col_scales[chunk * q.cols + col0 + c] = s;
  }
  __syncthreads();
  if (col >= q.cols) return;
  fp8b_emit<T, WHAT, E5M2>(q, t, row_f, col_f, row0, row_end, r_in, c_in, col, chunk);
}

// Rows alone: eight lanes a block of 128, sixteen numbers a lane, no shared memory; a warp four rows, two blocks of each.
// Bound by HBM: 8192 x 14336 bf16 60 us (5.9 TB/s).
template <class T, bool E5M2>
__global__ void __launch_bounds__(256) fp8b_quantize_rows_kernel(const Fp8bQuant q) {
  constexpr bool BF16 = sizeof(T) == 2;
  constexpr int U = 2;
  grid_dependency_wait();
  grid_launch_dependents();          // (products that read their weights meanwhile: altob200_fp8_block_gemm_args.b_ready)
  const int lane = threadIdx.x & 31;
  const int64_t col0 = (int64_t)blockIdx.x * (128 * U) + (lane & 7) * 16;
  for (int64_t at = blockIdx.y; at * 32 < q.rows; at += gridDim.y) {
    const int64_t row = at * 32 + (threadIdx.x >> 5) * 4 + (lane >> 3);
    const T* const x = static_cast<const T*>(q.x) + row * q.ld + col0;
    float v[U][16];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = row < q.rows && col0 + 128 * u < q.cols;      // (columns come in sixteens)
      if (BF16) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint4 w = in ? __ldg(reinterpret_cast<const uint4*>(x + 128 * u) + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            v[u][8 * k + 2 * j] = bf16lo_to_f32((&w.x)[j]);
            v[u][8 * k + 2 * j + 1] = bf16hi_to_f32((&w.x)[j]);
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 w = in ? __ldg(reinterpret_cast<const float4*>(x + 128 * u) + k) : make_float4(0, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[u][4 * k + j] = (&w.x)[j];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < 16; j += 2) m = absmax3_nan(m, v[u][j], v[u][j + 1]);
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
      const float s = fp8b_scale<E5M2>(m);
      const float2 f = fp8b_divisor(s);
      uint4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        (&w.x)[j] = fp8b_word<BF16, E5M2>(v[u][4 * j], v[u][4 * j + 1], v[u][4 * j + 2], v[u][4 * j + 3], f);
      const int64_t col = col0 + 128 * u;
      if (row < q.rows && col < q.cols) {
        *reinterpret_cast<uint4*>(q.row_codes + row * q.cols + col) = w;
        if ((lane & 7) == 0) q.row_scales[((int64_t)blockIdx.x * U + u) * q.rows + row] = s;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// values of codes and scales
// ---------------------------------------------------------------------------------------
// Eight codes of a row a thread.  Element (r, c): scales[(r >> row_shift) * row_stride + (c >> col_shift) * col_stride].
struct Fp8bDequant {
  const uint8_t* codes;
  const float* scales;
  int64_t rows, cols, row_stride, col_stride;
  int row_shift, col_shift;
  void* out;
};
template <bool E5M2, bool BF16>
__global__ void __launch_bounds__(256) fp8b_dequantize_kernel(const Fp8bDequant q) {
  grid_dependency_wait();
  const int64_t per_row = q.cols / 8, n = q.rows * per_row;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per_row, c = (i - r * per_row) * 8;
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(q.codes + r * q.cols + c));
    const float* s = q.scales + (r >> q.row_shift) * q.row_stride;
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 d = fp8x2_decode<E5M2>(((j < 2 ? w.x : w.y) >> (16 * (j & 1))) & 0xFFFFu);
      v[2 * j] = d.x;
      v[2 * j + 1] = d.y;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], __ldg(s + ((c + j) >> q.col_shift) * q.col_stride));
    if (BF16) {
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(q.out) + r * q.cols + c) =
          make_uint4(pack_bf16_rn(v[0], v[1]), pack_bf16_rn(v[2], v[3]), pack_bf16_rn(v[4], v[5]), pack_bf16_rn(v[6], v[7]));
    } else {
      float4* const o = reinterpret_cast<float4*>(static_cast<float*>(q.out) + r * q.cols + c);
      o[0] = make_float4(v[0], v[1], v[2], v[3]);
      o[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
}

// ---------------------------------------------------------------------------------------
// products of few rows
// ---------------------------------------------------------------------------------------
// Bound by the reading of B (the weights): every warp takes 16 NW of its rows as the 16-row side of the matrix instruction and
// rows of A as the 8-column side, in chunks of 128 of K that the CTA's eight warps share out; a chunk's products are
// scaled and added in fp32, the warps' sums joined through shared memory in their order.
// A lane's 16 bytes of a row are two instructions' operands: which of a chunk's numbers meet in one instruction does not
// matter as long as both sides agree, so nothing is shuffled.  FUSED: A is bf16 or fp32 and a lane makes the codes of the
// numbers that it needs, so that a token's step is one launch: 1 | 8 rows past 14336 x 4096 take 16.1 | 16.4 us (B alone 9.0), past
// 4096 x 4096 6.7 (2.6), 512 x 512 1.9.  (Codes that gemm_fp8_stream.cuh takes are faster there: this instruction converts
// both sides' 8 bits on every use.)
struct Fp8bRows {
  int64_t M, N, K;
  const void* a;         // codes [M, K], or numbers (FUSED, lda)
  int64_t lda;
  const uint8_t* b;      // codes [experts][N, K]
  const float *sa, *sb;
  int64_t sa_row, sa_chunk, sb_row, sb_chunk, sb_expert;
  int sa_shift, sb_shift;
  const int32_t* offs;
  int experts;
  int k_ranges;          // offs are rows of the reduced dimension (k_rows of them), every expert has an output of its own
  int64_t k_rows;
  int out_bf16;
  void* d;
  int64_t ldd;
};

template <bool E5M2>
__device__ __forceinline__ void fp8b_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (E5M2)
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e5m2.e5m2.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes of a row's 16 numbers at `at` and at `at` + 64 of a chunk, by the four lanes of the row; returns the scale.
template <class T, bool E5M2>
__device__ __forceinline__ float fp8b_row_codes(const T* row, int64_t k, int64_t K, bool there, uint4 (&w)[2]) {
  constexpr bool BF16 = sizeof(T) == 2;
  float v[32];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const bool in = there && k + 64 * h < K;
    if (BF16) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint4 u = in ? __ldg(reinterpret_cast<const uint4*>(row + k + 64 * h) + q) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[16 * h + 8 * q + 2 * j] = bf16lo_to_f32((&u.x)[j]);
          v[16 * h + 8 * q + 2 * j + 1] = bf16hi_to_f32((&u.x)[j]);
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 u = in ? __ldg(reinterpret_cast<const float4*>(row + k + 64 * h) + q) : make_float4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[16 * h + 4 * q + j] = (&u.x)[j];
      }
    }
  }
  float m = 0.0f;
#pragma unroll
  for (int j = 0; j < 16; ++j) m = absmax3_nan(m, v[2 * j], v[2 * j + 1]);
  m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
  m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
  const float s = fp8b_scale<E5M2>(m);
  const float2 f = fp8b_divisor(s);
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float* x = v + 16 * h + 4 * j;
      (&w[h].x)[j] = fp8b_word<BF16, E5M2>(x[0], x[1], x[2], x[3], f);
    }
  return s;
}

// T: the type of A's numbers, or uint8_t where A is codes.
template <class T, int NW, int J, bool E5M2>
__global__ void __launch_bounds__(256) fp8b_rows_kernel(const Fp8bRows q) {
  constexpr bool FUSED = sizeof(T) > 1;
  __shared__ float part[8][8 * J][16 * NW + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  grid_dependency_wait();
  const int64_t n0 = (int64_t)blockIdx.x * (16 * NW);
  int64_t row0 = 0, row1 = q.M, c0 = 0, c1 = (q.K + 127) / 128;
  const int e = (int)blockIdx.z;
  void* d = q.d;
  const int esz = q.out_bf16 ? 2 : 4;
  if (q.offs != nullptr && q.k_ranges) {
    // blocks of 128 from the expert's first row on, one run behind the other
    int64_t first = 0, end = 0;
    for (int i = 0; i <= e; ++i) {
      int64_t o = __ldg(q.offs + i);
      o = o < end ? end : o > q.k_rows ? q.k_rows : o;
      c0 = first;
      first += (o - end + 127) / 128;
      end = o;
    }
    c1 = first;
    d = static_cast<char*>(d) + (int64_t)e * q.M * q.ldd * esz;
  } else if (q.offs != nullptr) {
    // the running maximum of the ends (see Fp8bRun), so that no row has two experts: looked for by those that can have rows
    // (20 rows of 1500 experts of 48 x 144: 18 us, 32 where every one looks)
    const auto cut = [&](int o) { return o < 0 ? 0 : o > q.M ? (int)q.M : o; };
    const int end = e < q.experts ? cut(__ldg(q.offs + e)) : (int)q.M;
    int before = e > 0 ? cut(__ldg(q.offs + e - 1)) : 0;
    if (end <= before) return;
#pragma unroll 8
    for (int i = lane; i < e - 1; i += 32) before = max(before, cut(__ldg(q.offs + i)));
    row0 = __reduce_max_sync(0xFFFFFFFFu, before);
    row1 = end;
  }
  const bool zeros = e == q.experts;      // rows behind the last expert
  const uint8_t* const b = q.b + (q.k_ranges || zeros ? 0 : (int64_t)e * q.N * q.K);
  const float* const sb = q.sb + (q.k_ranges || zeros ? 0 : (int64_t)e * q.sb_expert);
  const uint8_t* bp[2 * NW];
  const float* sbp[2 * NW];
#pragma unroll
  for (int i = 0; i < 2 * NW; ++i) {
    const int64_t n = n0 + 8 * i + g < q.N ? n0 + 8 * i + g : q.N - 1;
    bp[i] = b + n * q.K;
    sbp[i] = sb + (n >> q.sb_shift) * q.sb_row;
  }
  for (int64_t m0 = row0 + (int64_t)blockIdx.y * (8 * J); m0 < row1; m0 += (int64_t)gridDim.y * (8 * J)) {
    float acc[NW][J][4];
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[w][j][i] = 0.0f;
    if (!zeros)
      for (int64_t c = c0 + warp; c < c1; c += 8) {
        const int64_t k = c * 128 + 16 * t;
        uint4 bw[2 * NW][2];
        float sw[2 * NW];
#pragma unroll
        for (int i = 0; i < 2 * NW; ++i) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            bw[i][h] = k + 64 * h < q.K ? __ldg(reinterpret_cast<const uint4*>(bp[i] + k + 64 * h)) : make_uint4(0, 0, 0, 0);
          sw[i] = __ldg(sbp[i] + c * q.sb_chunk);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int64_t m = m0 + 8 * j + g;
          const bool there = m < row1;
          uint4 aw[2];
          float s0, s1;
          if (FUSED) {
            const float s = fp8b_row_codes<T, E5M2>(static_cast<const T*>(q.a) + (there ? m : 0) * q.lda, k, q.K, there, aw);
            s0 = __shfl_sync(0xFFFFFFFFu, s, 8 * t);
            s1 = __shfl_sync(0xFFFFFFFFu, s, 8 * t + 4);
          } else {
            const uint8_t* const row = static_cast<const uint8_t*>(q.a) + (there ? m : 0) * q.K;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              aw[h] = there && k + 64 * h < q.K ? __ldg(reinterpret_cast<const uint4*>(row + k + 64 * h)) : make_uint4(0, 0, 0, 0);
            const int64_t ms = m0 + 8 * j + 2 * t;
            s0 = ms < row1 ? __ldg(q.sa + (ms >> q.sa_shift) * q.sa_row + c * q.sa_chunk) : 0.0f;
            s1 = ms + 1 < row1 ? __ldg(q.sa + ((ms + 1) >> q.sa_shift) * q.sa_row + c * q.sa_chunk) : 0.0f;
          }
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            float p[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint4 lo = bw[2 * w][h], hi = bw[2 * w + 1][h];
              fp8b_mma<E5M2>(p, lo.x, hi.x, lo.y, hi.y, aw[h].x, aw[h].y);
              fp8b_mma<E5M2>(p, lo.z, hi.z, lo.w, hi.w, aw[h].z, aw[h].w);
            }
            acc[w][j][0] = __fmaf_rn(p[0], __fmul_rn(sw[2 * w], s0), acc[w][j][0]);
            acc[w][j][1] = __fmaf_rn(p[1], __fmul_rn(sw[2 * w], s1), acc[w][j][1]);
            acc[w][j][2] = __fmaf_rn(p[2], __fmul_rn(sw[2 * w + 1], s0), acc[w][j][2]);
            acc[w][j][3] = __fmaf_rn(p[3], __fmul_rn(sw[2 * w + 1], s1), acc[w][j][3]);
          }
        }
      }
    __syncthreads();      // the sums of the rows before have been read
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[warp][8 * j + 2 * t + (i & 1)][16 * w + g + 8 * (i >> 1)] = acc[w][j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * J * 16 * NW; i += 256) {
      const int m = i / (16 * NW), n = i % (16 * NW);
      float s = part[0][m][n];
#pragma unroll
      for (int w = 1; w < 8; ++w) s += part[w][m][n];
      if (m0 + m < row1 && n0 + n < q.N) {
        const int64_t at = (m0 + m) * q.ldd + n0 + n;
        if (q.out_bf16) static_cast<__nv_bfloat16*>(d)[at] = __float2bfloat16_rn(s);
        else static_cast<float*>(d)[at] = s;
      }
    }
  }
}

static int sms() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  return n;
}

template <class T, int NW, int J>
static cudaError_t launch_rows(const Fp8bRows& q, dim3 grid, bool e5m2, cudaStream_t st) {
  return e5m2 ? launch_after(fp8b_rows_kernel<T, NW, J, true>, grid, dim3(256), 0, st, q)
              : launch_after(fp8b_rows_kernel<T, NW, J, false>, grid, dim3(256), 0, st, q);
}

static bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// in gemm_sm100.cu: the products of many rows
int fp8_block_gemm_tiles(const altob200_fp8_block_gemm_args* a, cudaStream_t st);
// and of few
int fp8_block_gemm_stream(const altob200_fp8_block_gemm_args* a, int64_t rows_a_run, cudaStream_t st);

}  // namespace altob200

using namespace altob200;

extern "C" {

int altob200_fp8_block_quantize(const altob200_fp8_block_quant_args* a, void* stream) {
  if (a == nullptr || a->rows < 0 || a->cols <= 0 || a->cols % 16 != 0 || a->ld < a->cols) return ALTOB200_EINVAL_SHAPE;
  if ((a->dtype != ALTOB200_DT_BF16 && a->dtype != ALTOB200_DT_F32) ||
      (a->format != ALTOB200_FMT_MXFP8_E4M3 && a->format != ALTOB200_FMT_MXFP8_E5M2))
    return ALTOB200_EUNSUPPORTED;
  if ((a->row_codes == nullptr) != (a->row_scales == nullptr) || (a->col_codes == nullptr) != (a->col_scales == nullptr) ||
      (a->row_codes == nullptr && a->col_codes == nullptr) || (a->offs != nullptr && a->experts <= 0))
    return ALTOB200_EINVAL_SHAPE;
  const int64_t esz = a->dtype == ALTOB200_DT_BF16 ? 2 : 4;
  if (off16(a->x) || (a->ld * esz) % 16 != 0 || off16(a->row_codes) || off16(a->col_codes) || (a->col_codes != nullptr && a->ld_col % 128 != 0))
    return ALTOB200_EINVAL_ALIGN;
  const int64_t chunks = a->offs != nullptr ? a->rows / 128 + a->experts : ceil_div(a->rows, 128);
  if (a->col_codes != nullptr && a->ld_col < chunks * 128) return ALTOB200_EINVAL_SHAPE;
  if (a->rows >= (1ll << 30)) return ALTOB200_ELIMIT;
  if (a->rows == 0) return ALTOB200_OK;
  if (a->x == nullptr) return ALTOB200_EINVAL_SHAPE;
  if (chunks > 65535 && a->col_codes != nullptr) return ALTOB200_ELIMIT;
  Fp8bQuant q = {a->x, a->rows, a->cols, a->ld, a->offs, a->experts, (uint8_t*)a->row_codes, a->row_scales, (uint8_t*)a->col_codes, a->ld_col,
                 a->col_scales, 0};
  const dim3 grid((unsigned)ceil_div(a->cols, 128), (unsigned)(chunks < 65535 ? chunks : 65535));
  const bool e5 = a->format == ALTOB200_FMT_MXFP8_E5M2;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t rc;
#define ALTOB200_Q(T, W) \
  rc = e5 ? launch_after(fp8b_quantize_kernel<T, W, true>, grid, dim3(256), 0, st, q) : launch_after(fp8b_quantize_kernel<T, W, false>, grid, dim3(256), 0, st, q)
  if (a->col_codes == nullptr) {
    const int64_t groups = ceil_div(a->rows, 32);
    const dim3 g((unsigned)ceil_div(a->cols, 256), (unsigned)(groups < 65535 ? groups : 65535));
#define ALTOB200_QR(T) \
  rc = e5 ? launch_after(fp8b_quantize_rows_kernel<T, true>, g, dim3(256), 0, st, q) : launch_after(fp8b_quantize_rows_kernel<T, false>, g, dim3(256), 0, st, q)
    if (a->dtype == ALTOB200_DT_BF16) { ALTOB200_QR(__nv_bfloat16); }
    else { ALTOB200_QR(float); }
#undef ALTOB200_QR
  } else if (a->dtype == ALTOB200_DT_BF16) {
    if (a->row_codes == nullptr) { ALTOB200_Q(__nv_bfloat16, FP8B_COLS); }
    else { ALTOB200_Q(__nv_bfloat16, (FP8B_ROWS | FP8B_COLS)); }
  } else {
    if (a->row_codes == nullptr) { ALTOB200_Q(float, FP8B_COLS); }
    else { ALTOB200_Q(float, (FP8B_ROWS | FP8B_COLS)); }
  }
  return rc == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

int altob200_fp8_block_quantize_squares(const void* x, int32_t dtype, int32_t format, int64_t matrices, int64_t rows, int64_t cols, int64_t ld,
                                        int64_t matrix_stride, void* codes, void* codes_t, float* scales, void* stream) {
  if (matrices < 0 || rows <= 0 || cols <= 0 || cols % 16 != 0 || rows % 16 != 0 || ld < cols) return ALTOB200_EINVAL_SHAPE;
  if ((dtype != ALTOB200_DT_BF16 && dtype != ALTOB200_DT_F32) || (format != ALTOB200_FMT_MXFP8_E4M3 && format != ALTOB200_FMT_MXFP8_E5M2))
    return ALTOB200_EUNSUPPORTED;
  const int64_t esz = dtype == ALTOB200_DT_BF16 ? 2 : 4;
  if (off16(x) || (ld * esz) % 16 != 0 || (matrix_stride * esz) % 16 != 0 || off16(codes) || off16(codes_t)) return ALTOB200_EINVAL_ALIGN;
  if (ceil_div(rows, 128) > 65535 || matrices > 65535 || rows >= (1ll << 30)) return ALTOB200_ELIMIT;
  if (matrices == 0) return ALTOB200_OK;
  if (x == nullptr || scales == nullptr || (codes == nullptr && codes_t == nullptr)) return ALTOB200_EINVAL_SHAPE;
  Fp8bQuant q = {x, rows, cols, ld, nullptr, 0, (uint8_t*)codes, scales, (uint8_t*)codes_t, rows, nullptr, matrix_stride};
  const dim3 grid((unsigned)ceil_div(cols, 128), (unsigned)ceil_div(rows, 128), (unsigned)matrices);
  const bool e5 = format == ALTOB200_FMT_MXFP8_E5M2;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t rc;
  if (dtype == ALTOB200_DT_BF16) { ALTOB200_Q(__nv_bfloat16, FP8B_SQUARES); }
  else { ALTOB200_Q(float, FP8B_SQUARES); }
#undef ALTOB200_Q
  return rc == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

int altob200_fp8_block_dequantize(const void* codes, int32_t format, int64_t rows, int64_t cols, const altob200_fp8_block_scale* scale,
                                  int32_t out_dtype, void* out, void* stream) {
  if (rows < 0 || cols <= 0 || cols % 8 != 0 || scale == nullptr) return ALTOB200_EINVAL_SHAPE;
  if ((format != ALTOB200_FMT_MXFP8_E4M3 && format != ALTOB200_FMT_MXFP8_E5M2) || (out_dtype != ALTOB200_DT_BF16 && out_dtype != ALTOB200_DT_F32))
    return ALTOB200_EUNSUPPORTED;
  if ((scale->row_shift != 0 && scale->row_shift != 7) || (scale->chunk_shift != 0 && scale->chunk_shift != 7)) return ALTOB200_EINVAL_SHAPE;
  if (rows == 0) return ALTOB200_OK;
  if (codes == nullptr || out == nullptr || scale->scales == nullptr) return ALTOB200_EINVAL_SHAPE;
  if ((reinterpret_cast<uintptr_t>(codes) & 7) || off16(out)) return ALTOB200_EINVAL_ALIGN;
  Fp8bDequant q = {(const uint8_t*)codes, scale->scales, rows, cols, scale->row_stride, scale->chunk_stride, scale->row_shift, scale->chunk_shift, out};
  int64_t blocks = ceil_div(rows * (cols / 8), 256);
  const int64_t most = (int64_t)sms() * 16;
  if (blocks > most) blocks = most;
  const bool e5 = format == ALTOB200_FMT_MXFP8_E5M2, bf = out_dtype == ALTOB200_DT_BF16;
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)blocks), block(256);
  const cudaError_t rc = e5 ? (bf ? launch_after(fp8b_dequantize_kernel<true, true>, grid, block, 0, st, q) : launch_after(fp8b_dequantize_kernel<true, false>, grid, block, 0, st, q))
                            : (bf ? launch_after(fp8b_dequantize_kernel<false, true>, grid, block, 0, st, q) : launch_after(fp8b_dequantize_kernel<false, false>, grid, block, 0, st, q));
  return rc == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

int altob200_fp8_block_gemm(const altob200_fp8_block_gemm_args* a, void* stream) {
  if (a == nullptr || a->M < 0 || a->N <= 0 || a->K < 0 || a->K % 16 != 0 || a->ldd < a->N) return ALTOB200_EINVAL_SHAPE;
  if (a->format != ALTOB200_FMT_MXFP8_E4M3 && a->format != ALTOB200_FMT_MXFP8_E5M2) return ALTOB200_EUNSUPPORTED;
  if (a->mode < 0 || a->mode > 2 || (a->mode != 0 && (a->offs == nullptr || a->experts <= 0))) return ALTOB200_EINVAL_SHAPE;
  const bool numbers = a->a_dtype == ALTOB200_DT_BF16 || a->a_dtype == ALTOB200_DT_F32;
  if (!numbers && a->a_dtype != -1) return ALTOB200_EUNSUPPORTED;
  if (numbers && a->mode == 2) return ALTOB200_EUNSUPPORTED;
  if (a->out_dtype != ALTOB200_DT_BF16 && a->out_dtype != ALTOB200_DT_F32) return ALTOB200_EUNSUPPORTED;
  if ((a->sa.row_shift != 0 && a->sa.row_shift != 7) || (a->sb.row_shift != 0 && a->sb.row_shift != 7)) return ALTOB200_EINVAL_SHAPE;
  const int64_t esz = a->out_dtype == ALTOB200_DT_BF16 ? 2 : 4;
  if (a->N % 16 != 0 || (a->mode == 2 && (a->k_rows < 0 || a->K < (a->k_rows / 128 + a->experts) * 128))) return ALTOB200_EINVAL_SHAPE;
  if (off16(a->a) || off16(a->b) || off16(a->d) || (a->ldd * esz) % 16 != 0) return ALTOB200_EINVAL_ALIGN;
  if (numbers && ((a->lda * (a->a_dtype == ALTOB200_DT_BF16 ? 2 : 4)) % 16 != 0 || a->lda < a->K)) return ALTOB200_EINVAL_ALIGN;
  if (a->M >= (1ll << 30) || a->N >= (1ll << 30) || a->K >= (1ll << 30) || a->experts > 32767) return ALTOB200_ELIMIT;
  if (a->M == 0) return ALTOB200_OK;
  if (a->d == nullptr || (a->K > 0 && (a->a == nullptr || a->b == nullptr || a->sb.scales == nullptr || (!numbers && a->sa.scales == nullptr))))
    return ALTOB200_EINVAL_SHAPE;
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t per_run = a->mode == 1 ? ceil_div(a->M, a->experts) : a->M;
  int done = fp8_block_gemm_stream(a, per_run, st);
  if (done == ALTOB200_EUNSUPPORTED && !numbers) done = fp8_block_gemm_tiles(a, st);
  if (done != ALTOB200_EUNSUPPORTED) return done;
  Fp8bRows q;
  q.M = a->M; q.N = a->N; q.K = a->K;
  q.a = a->a; q.lda = a->lda; q.b = (const uint8_t*)a->b;
  q.sa = a->sa.scales; q.sa_row = a->sa.row_stride; q.sa_chunk = a->sa.chunk_stride; q.sa_shift = a->sa.row_shift;
  q.sb = a->sb.scales; q.sb_row = a->sb.row_stride; q.sb_chunk = a->sb.chunk_stride; q.sb_shift = a->sb.row_shift; q.sb_expert = a->sb.expert_stride;
  q.offs = a->mode == 0 ? nullptr : a->offs;
  q.experts = a->mode == 0 ? 1 : a->experts;
  q.k_ranges = a->mode == 2;
  q.k_rows = a->k_rows;
  q.out_bf16 = a->out_dtype == ALTOB200_DT_BF16;
  q.d = a->d; q.ldd = a->ldd;
  const bool e5 = a->format == ALTOB200_FMT_MXFP8_E5M2;
  const bool wide = ceil_div(a->N, 32) * (a->mode == 0 ? 1 : a->experts) >= 2 * sms();
  const int tokens = numbers ? 8 : 32;
  int64_t y = ceil_div(per_run, tokens);
  if (y > 65535) y = 65535;
  const dim3 grid((unsigned)ceil_div(a->N, wide ? 32 : 16), (unsigned)y, (unsigned)(a->mode == 1 ? a->experts + 1 : q.experts));
  cudaError_t rc;
#define ALTOB200_R(T, J) rc = wide ? launch_rows<T, 2, J>(q, grid, e5, st) : launch_rows<T, 1, J>(q, grid, e5, st)
  if (!numbers) { ALTOB200_R(uint8_t, 4); }
  else if (a->a_dtype == ALTOB200_DT_BF16) { ALTOB200_R(__nv_bfloat16, 1); }
  else { ALTOB200_R(float, 1); }
#undef ALTOB200_R
  return rc == cudaSuccess ? ALTOB200_OK : ALTOB200_ECUDA;
}

}  // extern "C"
