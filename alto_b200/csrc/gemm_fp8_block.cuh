// FP8 GEMM with one fp32 scale for each block of 128 along K, for sm_100a.
//
//   D[m, n] = sum over chunks c of 128 along K of sa[m, c] * sb[n, c] * sum_{k in c} A[m, k] * B[n, k]
//
// The scales are fp32, so they cannot ride on a block-scaled MMA (8-bit scales): the tensor cores sum one chunk at a time
// into tensor memory and CUDA cores add it, times both scales, to the fp32 result in registers.
//
// A cluster of two CTAs owns 256 x 256 of the output (cta_group::2), each CTA 128 rows of it; 384 threads a CTA:
//   warp 0      producer: per chunk (128 bytes of K) this CTA's 128 rows of A and its half of B's 256 by TMA; and the rows'
//               factors (sa, times sb where one serves 128 columns) into a ring in shared memory, loaded two chunks ahead
//   warp 1      MMA issuer (leader): per chunk two times four tcgen05.mma of 256 x 128 x 32, into four accumulators of 128
//               columns (two chunks), which are all of the tensor memory
//   warp 2      waits for the issuer (as in the block-scaled pair kernel)
//   warp 3      the list of units; then waits for the fold warps and releases them at named barriers
//   warps 4-11  fold: per tensor-memory lane quarter two warps of 32 rows x 128 columns, the sums in 128 registers a lane.
//               64 columns of a chunk at a time come into registers; the accumulator is given back when the last have.
// Rows of A may belong to experts in runs of any length (mode 1): a unit of 256 rows begins at a run's first row, rows of the
// next run that a tile holds beyond its own are multiplied by the wrong weights and not stored.  In mode 2 the reduced
// dimension is cut into the experts' runs of whole chunks.
//
// What bounds it: with the fold's arithmetic left out a chunk takes 630 to 720 cycles (512 of them MMAs; the operand bytes
// in and out of shared memory are most of the rest), with it 835 to 870, with a factor for every column 1040 to 1080: the
// multiply-adds of a chunk take 280 (560 with the column factors' products) on every scheduler, and the way of a chunk
// through a fold warp is wait, 64 columns out of tensor memory, their multiply-adds, 64 more.  The clock falls with the power
// (1.4 to 1.6 GHz), so times vary with what ran before: 8192 x 4096 x 14336 and the two others of a training step
// 445 / 432 / 530 to 650 us.  Before, in cycles a chunk (one factor / one a column): 1040 / 1400 with instructions of 256
// columns in two accumulators, which the issuer waits for longer; 1180 / 1240 with the scales loaded by the fold warps (in registers, where
// a spilled one costs more than the load); 960 / 1310 with them by cp.async; 1330 / 1080 with the factors made by the waiting
// warp; 905 / 1230 with fold warps that look at the barriers themselves.  A column factor in the 16 x 128-bit layout (eight
// shared-memory words a lane and 32 columns instead of 32) 2000.  Sixteen fold warps of 64 columns instead of eight of 128: 16 to
// 45 % more a chunk (2048 x 2048, 0.50 us for 0.43, 0.75 for 0.57).  A launch of one chunk a tile takes 7.8 us (2048 x 2048 bf16): some
// 0.7 to begin, 2.4 to the first chunk (most of it the fetch of instructions that no SM has yet: copies issued before the factors'
// loads, and prefetched descriptors, took as long or longer), 2.5 for the stores and the end.
#pragma once
// (included by gemm_sm100.cu inside namespace altob200, after the kernels it shares helpers with)

struct F8Args {
  int64_t M, N, K;
  const float *sa, *sb;
  int64_t sa_row, sa_chunk, sb_row, sb_chunk, sb_expert;
  int sa_shift;
  const int32_t* offs;
  int mode, experts;
  int64_t k_rows;
  int row_base;            // mode 1: of the experts' rows, those in front of A's
  void* d;
  int64_t ldd;
  int tiles_n, group_m;
  uint32_t idesc;
  uint64_t wait_ns;
};

struct CfgF8 {
  static constexpr int THREADS = 384;
  static constexpr int BN = 256;
  static constexpr int A_BYTES = BM * STAGE_K_BYTES;
  static constexpr int B_BYTES = (BN / 2) * STAGE_K_BYTES;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int FOLD_WARPS = 8;
  static constexpr int EPI_BYTES = FOLD_WARPS * 8192;      // 32 rows x 128 bytes a warp, twice
  // Rings of B's column factors and of the rows' factors [half][row], one slot a chunk.  A slot is written again when the MMAs
  // of the chunk STAGES before have finished; these began when the chunk two before them had been read out by every fold
  // warp, which reads a chunk out only after it has added the one before.
  static constexpr int FAC = 8;
  static constexpr int FAC_BYTES = FAC * BN * 4;
  static constexpr int ROW_FAC = FAC;
  static constexpr int ROW_FAC_BYTES = ROW_FAC * 256 * 4;
  static constexpr int MAX_UNITS = 4096, MAX_RUNS = 1024;  // of a launch
  // column factors (a scale for every row of B, no units), or units; and runs
  static constexpr int EXTRA_BYTES = MAX_UNITS * 4 > FAC_BYTES ? MAX_UNITS * 4 : FAC_BYTES;
  static constexpr int RUN_BYTES = 16 + MAX_RUNS * 4;      // (counts in front)
  static constexpr int NUM_BARS = 2 * STAGES + 8 + FAC + 1;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + EXTRA_BYTES + RUN_BYTES + ROW_FAC_BYTES + 1024 /*align*/ + 512 /*barriers*/;
  static_assert(NUM_BARS * 8 + 64 <= 512, "barrier area");
  static_assert(SMEM_BYTES <= 232448, "shared memory budget");
  // setmaxnreg.inc takes only what setmaxnreg.dec released of the registers at launch
  static constexpr int REGS_LAUNCH = 168, REGS_SMALL = 56, REGS_FOLD = 224;
  static_assert(128 * REGS_SMALL + 256 * REGS_FOLD <= THREADS * REGS_LAUNCH, "setmaxnreg budget");
};

__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// An arrival by one lane of a converged warp, without a branch.
__device__ __forceinline__ void mbar_arrive_cluster_one(uint32_t cluster_addr) {
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\t"
      "@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}"
      ::"r"(cluster_addr)
      : "memory");
}
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// A wait for copies that are on their way when a role has given up: a millisecond at least, however short the others' limit is.
__device__ __forceinline__ uint64_t drain_limit(uint64_t limit) { return limit > (1ull << 21) ? limit : 1ull << 21; }
// The operand copies of a CTA pair that are on their way when a role has given up land before the CTAs end.  The leader's producer
// issued `mine` stages, the peer's `theirs`; a stage goes out when the one STAGES before has been consumed in both, so that only the
// last STAGES can be on their way.  A stage's bytes complete on the leader's barrier, which expects those of both: where one did
// not issue it, the leader makes up for that.  By one warp of the leader; once a wait has run out, the later ones have waited as long.
template <int STAGES, int STAGE_BYTES>
__device__ __forceinline__ void drain_pair(uint64_t* full_bar, uint32_t mine, uint32_t theirs, int lane, uint32_t never, uint64_t limit) {
  const uint32_t most = mine > theirs ? mine : theirs;
  bool landed = true;
  for (uint32_t i = most < STAGES ? 0 : most - STAGES; i < most && landed; ++i) {
    uint64_t* const bar = &full_bar[i % STAGES];
    if (lane == 0) {
      if (i >= mine) mbar_expect_tx(bar, STAGE_BYTES);
      else if (i >= theirs) mbar_complete_tx(bar, STAGE_BYTES);
    }
    __syncwarp();
    landed = __all_sync(0xFFFFFFFFu, mbar_wait_tight(smem_u32(bar), (i / STAGES) & 1u, never, limit));
  }
}
// The same of a ring of a CTA's own barriers, whose last `issued` phases were all armed.
template <int SLOTS>
__device__ __forceinline__ void drain_ring(uint64_t* bars, uint32_t issued, uint32_t never, uint64_t limit) {
  bool landed = true;
  for (uint32_t i = issued < SLOTS ? 0 : issued - SLOTS; i < issued && landed; ++i)
    landed = __all_sync(0xFFFFFFFFu, mbar_wait_tight(smem_u32(&bars[i % SLOTS]), (i / SLOTS) & 1u, never, limit));
}
__device__ __forceinline__ uint32_t thread_here() {      // (not kept in a register from elsewhere)
  uint32_t v;
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(v));
  return v;
}
// The 32 values in r have landed (tcgen05.wait::ld came before): nothing that uses them can move above this.
__device__ __forceinline__ void tc_landed32(uint32_t* r) {
#define ALTOB200_RW8(o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
  asm volatile("" : ALTOB200_RW8(0), ALTOB200_RW8(8), ALTOB200_RW8(16), ALTOB200_RW8(24));
#undef ALTOB200_RW8
}

// 32 columns of a warp's rows, a row a lane: acc += r * f (one B factor, in f already), or r * f * column factor.
template <bool B_ROWS>
__device__ __forceinline__ void f8_fold(float2* acc, const uint32_t* r, float f, uint32_t fcol) {
  const float2 f2 = make_float2(f, f);
  if constexpr (!B_ROWS) {
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[j] = __ffma2_rn(make_float2(u2f(r[2 * j]), u2f(r[2 * j + 1])), f2, acc[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 w = ld_shared_f32x4(fcol + 16u * j);
      const float2 w0 = __fmul2_rn(f2, make_float2(w.x, w.y)), w1 = __fmul2_rn(f2, make_float2(w.z, w.w));
      acc[2 * j] = __ffma2_rn(make_float2(u2f(r[4 * j]), u2f(r[4 * j + 1])), w0, acc[2 * j]);
      acc[2 * j + 1] = __ffma2_rn(make_float2(u2f(r[4 * j + 2]), u2f(r[4 * j + 3])), w1, acc[2 * j + 1]);
    }
  }
}

struct F8Tile {
  int row0, row_end;       // of A: the tile's first one, the end of its run
  int nb, expert, batch;
  int chunk0, chunks;      // along K
};

// mode 1: units (expert << 16 | unit of the run) and runs' first rows; mode 2: the runs' first chunks.
// Shared-memory addresses (one register for all): counts (units, tiles), units, runs.
struct F8Lists {
  uint32_t at;
  __device__ __forceinline__ uint32_t word(uint32_t i) const {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at + 4u * i));
    return v;
  }
  __device__ __forceinline__ uint32_t n_units() const { return word(0); }
  __device__ __forceinline__ uint32_t n_tiles() const { return word(1); }
  __device__ __forceinline__ uint32_t run(uint32_t i) const { return word(4 + i); }
  __device__ __forceinline__ uint32_t unit(uint32_t i) const { return word(4 + CfgF8::MAX_RUNS + i); }
};

// x / d; inv: 1 / d rounded.  (A tile's coordinates are on every role's way from one tile to the next.)
__device__ __forceinline__ uint32_t f8_div(uint32_t x, uint32_t d, float inv) {
  if (x >= (1u << 20)) return x / d;
  uint32_t q = (uint32_t)__fmul_rz((float)x, inv);
  const int r = (int)(x - q * d);
  q += r >= (int)d ? 1u : 0u;
  q -= r < 0 ? 1u : 0u;
  return q;
}
__device__ __forceinline__ F8Tile f8_tile(const F8Args& a, const F8Lists& l, uint32_t tile) {
  F8Tile t;
  t.batch = 0;
  t.expert = 0;
  t.chunk0 = 0;
  t.chunks = (int)((a.K + 127) >> 7);
  const uint32_t tiles_n = (uint32_t)a.tiles_n;
  const uint32_t units = a.mode == 1 ? l.n_units() : (uint32_t)((a.M + 255) >> 8);
  if (a.mode == 2) {
    const uint32_t per = units * tiles_n;
    t.batch = (int)f8_div(tile, per, __frcp_rn((float)per));
    tile -= (uint32_t)t.batch * per;
    t.chunk0 = (int)l.run(t.batch);
    t.chunks = (int)l.run(t.batch + 1) - t.chunk0;
  }
  // groups of group_m units swept across all columns, the unit running fastest: a group's rows of A stay in L2
  const uint32_t gm = (uint32_t)a.group_m, per_group = gm * tiles_n;
  const uint32_t g = f8_div(tile, per_group, __frcp_rn((float)per_group)), in = tile - g * per_group;
  const uint32_t left = units - g * gm, rows = left < gm ? left : gm;
  const uint32_t nb = f8_div(in, rows, __frcp_rn((float)rows)), u = g * gm + in - nb * rows;
  t.nb = (int)nb;
  if (a.mode == 1) {
    const uint32_t w = l.unit(u);
    t.expert = (int)(w >> 16);
    t.row0 = (int)(l.run(t.expert) + (w & 0xFFFFu) * 256u);
    t.row_end = (int)l.run(t.expert + 1);
    if (t.expert == a.experts) t.chunks = 0;      // rows behind the last run
  } else {
    t.row0 = (int)(u * 256u);
    t.row_end = (int)a.M;
  }
  return t;
}

// The lists, by one warp; returns the number of units.
__device__ __forceinline__ int f8_lists(const F8Args& a, int lane, uint32_t* units, uint32_t* runs) {
  int64_t limit = a.mode == 1 ? a.M : a.k_rows;
  const int total = a.experts + (a.mode == 1 ? 1 : 0);
  const int size = a.mode == 1 ? 256 : 128;
  int carry_end = 0, carry = 0;
  for (int e0 = 0; e0 < total; e0 += 32) {
    const int e = e0 + lane;
    int end = e < a.experts ? max(__ldg(a.offs + e), 0) - a.row_base : e == a.experts ? (int)limit : 0;
    end = end < 0 ? 0 : (int64_t)end > limit ? (int)limit : end;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, end, d);
      if (lane >= d && o > end) end = o;
    }
    if (end < carry_end) end = carry_end;
    int start = __shfl_up_sync(0xFFFFFFFFu, end, 1);
    if (lane == 0) start = carry_end;
    if (e >= total) start = end;
    const int n = (end - start + size - 1) / size;
    int sum = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xFFFFFFFFu, sum, d);
      if (lane >= d) sum += o;
    }
    const int before = carry + sum - n;
    if (e < total) runs[e] = a.mode == 1 ? (uint32_t)start : (uint32_t)before;
    if (a.mode == 1)
      for (int i = 0; i < n; ++i) units[before + i] = ((uint32_t)e << 16) | (uint32_t)i;
    carry_end = __shfl_sync(0xFFFFFFFFu, end, 31);
    carry = __shfl_sync(0xFFFFFFFFu, before + n, 31);
  }
  if (lane == 0) runs[total] = a.mode == 1 ? (uint32_t)limit : (uint32_t)carry;
  return carry;
}

// B_ROWS: a scale for every row of B (columns of the output), else for 128 of them.
template <bool OUT_BF16, bool B_ROWS>
__global__ void __launch_bounds__(CfgF8::THREADS, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                      const __grid_constant__ CUtensorMap tmap_d, const F8Args args) {
  using C = CfgF8;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi = smem + C::STAGES * C::STAGE_BYTES;
  float* row_fac = reinterpret_cast<float*>(epi + C::EPI_BYTES);
  uint32_t* counts = reinterpret_cast<uint32_t*>(epi + C::EPI_BYTES + C::ROW_FAC_BYTES);
  uint32_t* runs = counts + 4;
  uint32_t* units = runs + C::MAX_RUNS;
  float* fac = reinterpret_cast<float*>(units);
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + C::EPI_BYTES + C::ROW_FAC_BYTES + C::EXTRA_BYTES + C::RUN_BYTES);
  uint64_t* full_bar = bars;                      // leader: operand bytes of both CTAs
  uint64_t* empty_bar = bars + C::STAGES;         // each CTA, by the leader's commit
  uint64_t* acc_full = bars + 2 * C::STAGES;      // each CTA, by the leader's commit [chunk & 1]
  uint64_t* acc_empty = acc_full + 4;             // leader: the fold warps of both CTAs
  uint64_t* fac_full = acc_empty + 4;             // each CTA: bytes of its own factors
  uint64_t* mma_done = fac_full + C::FAC;         // each CTA, where a role has given up: by the leader's last commit
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* never = abort_flag + 1;           // an abort flag that nothing raises
  volatile uint32_t* ends = reinterpret_cast<volatile uint32_t*>(never + 1);   // stages issued here; by the peer: its own, its abort flag

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();        // 0 = leader
  const bool leader = rank == 0;
  const uint32_t pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], C::FOLD_WARPS);
    }
    for (int f = 0; f < C::FAC; ++f) mbar_init(&fac_full[f], B_ROWS ? 2 : 1);
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    *never = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();   // the peer's barriers are initialised before anything can arrive on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
  const uint64_t limit = args.wait_ns * 2ull;     // cycles, see the waits
  grid_dependency_wait();
  if (warp == 3) {
    uint32_t n_tiles = (uint32_t)((args.M + 255) >> 8) * (uint32_t)args.tiles_n, n = 0;
    if (args.mode != 0) {
      n = (uint32_t)f8_lists(args, lane, units, runs);
      n_tiles = args.mode == 1 ? n * (uint32_t)args.tiles_n : n_tiles * (uint32_t)args.experts;
    }
    if (lane == 0) {
      counts[0] = n;
      counts[1] = n_tiles;
    }
  }
  __syncthreads();
  const F8Lists lists = {smem_u32(counts)};

  if (warp < 4) {
    setmaxnreg_dec<C::REGS_SMALL>();
    const uint32_t n_tiles = lists.n_tiles();
    if (warp == 0) {
      // ------------------------------ producer ------------------------------
      // Also leaves the rows' factors of every chunk in shared memory, loaded two chunks ahead.
      struct Scales {
        float a[4], b[2];
      } q[2];
      uint32_t f_tile_at = pair;    // of the factors: next tile
      int f_left = 0;
      int at_a[4] = {0, 0, 0, 0}, at_b[2] = {0, 0};      // (fewer than 2^31 scales)
      auto request = [&](Scales& v) {
        while (f_left == 0) {
          if (f_tile_at >= n_tiles) return;
          const F8Tile t = f8_tile(args, lists, f_tile_at);
          f_tile_at += n_pairs;
          f_left = t.chunks;
          if (f_left == 0) continue;
          const int row0 = t.row0 + (int)rank * BM + lane, last = (int)args.M - 1;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            at_a[i] = ((row0 + 32 * i < last ? row0 + 32 * i : last) >> args.sa_shift) * (int)args.sa_row + t.chunk0 * (int)args.sa_chunk;
          if (!B_ROWS) {
            const int blocks = (int)((args.N + 127) >> 7);
#pragma unroll
            for (int h = 0; h < 2; ++h)
              at_b[h] = t.expert * (int)args.sb_expert + (t.nb * 2 + h < blocks ? t.nb * 2 + h : blocks - 1) * (int)args.sb_row + t.chunk0 * (int)args.sb_chunk;
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v.a[i] = __ldg(args.sa + at_a[i]);
          at_a[i] += (int)args.sa_chunk;
        }
        if (!B_ROWS) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            v.b[h] = __ldg(args.sb + at_b[h]);
            at_b[h] += (int)args.sb_chunk;
          }
        }
        --f_left;
      };
      auto leave = [&](const Scales& v, uint32_t slot) {
        float* const at = row_fac + slot * 256 + lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (B_ROWS) {
            at[32 * i] = v.a[i];
          } else {
            at[32 * i] = __fmul_rn(v.a[i], v.b[0]);
            at[128 + 32 * i] = __fmul_rn(v.a[i], v.b[1]);
          }
        }
        __syncwarp();
        mbar_arrive_lane0(smem_u32(&fac_full[slot]), lane);
      };
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) q[i].a[j] = q[i].b[j >> 1] = 0.0f;
      request(q[0]);
      request(q[1]);
      const bool elected = elect_one();
      uint32_t s = 0, phase = 1, slot = 0, tile = pair, stages = 0;
      int left = 0;
      int32_t kx = 0, ya = 0, yb = 0;
      uint32_t fac_bytes = 0;
      const float* sb_at = nullptr;
      bool alive = true, more = true;
      while (more && alive) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          while (left == 0 && more) {
            more = tile < n_tiles;
            if (!more) break;
            const F8Tile t = f8_tile(args, lists, tile);
            tile += n_pairs;
            left = t.chunks;
            kx = t.chunk0 * 128;
            ya = t.row0 + (int32_t)rank * BM;
            yb = (int32_t)((args.mode == 1 ? (int64_t)t.expert * args.N : 0) + (int64_t)t.nb * C::BN + (int64_t)rank * (C::BN / 4));
            if (B_ROWS) {
              const int64_t n0 = (int64_t)t.nb * C::BN;
              fac_bytes = (uint32_t)(args.N - n0 < C::BN ? args.N - n0 : C::BN) * 4u;
              sb_at = args.sb + (int64_t)t.chunk0 * args.sb_chunk + n0;
            }
          }
          if (!more) break;
          alive = __all_sync(0xFFFFFFFFu, mbar_wait_tight(smem_u32(&empty_bar[s]), phase, abort_addr, limit));
          if (!alive) break;
          uint8_t* st = smem + s * C::STAGE_BYTES;
          if (elected) {
            if (leader) mbar_expect_tx(&full_bar[s], 2 * C::STAGE_BYTES);
            const uint32_t full_leader = mapa_u32(smem_u32(&full_bar[s]), 0);
            tma_load_2d_pair(st, &tmap_a, kx, ya, full_leader);
            tma_load_2d_pair(st + C::A_BYTES, &tmap_b, kx, yb, full_leader);
            tma_load_2d_pair(st + C::A_BYTES + C::B_BYTES / 2, &tmap_b, kx, yb + C::BN / 2, full_leader);
            if (B_ROWS) {
              mbar_expect_tx(&fac_full[slot], fac_bytes);
              bulk_load(fac + slot * C::BN, sb_at, fac_bytes, &fac_full[slot]);
            }
          }
          __syncwarp();
          leave(q[i], slot);
          request(q[i]);
          kx += 128;
          if (B_ROWS) sb_at += args.sb_chunk;
          --left;
          ++stages;
          if (++slot == C::FAC) slot = 0;
          if (++s == C::STAGES) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
      if (!alive) report_timeout(abort_flag, 31);
      if (lane == 0) ends[0] = stages;
    } else if (warp == 1) {
      // ------------------------------ MMA issuer (leader) ------------------------------
      if (leader) {
        const bool elected = elect_one();
        uint32_t s = 0, buf = 0;
        bool alive = true;
        const uint32_t smem_base = smem_u32(smem);
        for (uint32_t tile = pair; tile < n_tiles && alive; tile += n_pairs) {
          const F8Tile t = f8_tile(args, lists, tile);
          for (int c = 0; c < t.chunks; ++c) {
            const int64_t left = args.K - (int64_t)(t.chunk0 + c) * 128;
            const int n_mma = left >= 128 ? 4 : (int)((left + 31) / 32);
            const uint32_t a_lo = ((smem_base + s * C::STAGE_BYTES) >> 4) | 0x10000u, b_lo = a_lo + (C::A_BYTES >> 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              alive = alive && !named_barrier_or(1 + h, 64, false);
              if (!alive) break;
              tc_fence_after();
              if (elected) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                  if (j < n_mma)
                    tc_mma_f8_pair(tmem_base + buf * C::BN + h * 128, desc_of(DESC_SW128_HI, a_lo + 2 * j),
                                   desc_of(DESC_SW128_HI, b_lo + h * (C::B_BYTES >> 5) + 2 * j), args.idesc, (uint32_t)j);
                if (h == 1) tc_commit_pair(&empty_bar[s]);
                tc_commit_pair(&acc_full[2 * buf + h]);
              }
              __syncwarp();
            }
            if (!alive) break;
            buf ^= 1u;
            if (++s == C::STAGES) s = 0;
          }
        }
      }
    } else if (warp == 2) {
      // ------------------------------ wait warp (leader) ------------------------------
      if (leader) {
        uint32_t s = 0, phase = 0, chunk = 0;
        bool alive = true;
        for (uint32_t tile = pair; tile < n_tiles && alive; tile += n_pairs) {
          const F8Tile t = f8_tile(args, lists, tile);
          for (int c = 0; c < t.chunks; ++c, ++chunk) {
            // the accumulator's chunk before has been read out, the operands are there
            const uint32_t full = smem_u32(&full_bar[s]), gone_phase = ((chunk >> 1) & 1) ^ 1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t gone = smem_u32(&acc_empty[2 * (chunk & 1) + h]);
              const bool ok = alive && mbar_wait3_tight(full, full, phase, gone, gone_phase, abort_addr, limit);
              if (alive && named_barrier_or(1 + h, 64, !ok)) {
                alive = false;
                report_timeout(abort_flag, !mbar_complete(gone, gone_phase) ? 32 : 33);
              }
            }
            if (!alive) break;
            if (++s == C::STAGES) {
              s = 0;
              phase ^= 1u;
            }
          }
        }
      }
    } else {
      // ------------------------------ wait warp of the fold ------------------------------
      // Looks at the barriers for the fold warps and releases them, a group each, at named barriers 3 and 4 (a raised
      // predicate: a failure).
      uint32_t chunk = 0, told = 0;          // told: groups that know of a failure (and have left)
      bool alive = true;
      for (uint32_t tile = pair; tile < n_tiles && told != 3u; tile += n_pairs) {
        const int chunks = f8_tile(args, lists, tile).chunks;
        for (int c = 0; c < chunks && told != 3u; ++c, ++chunk) {
          const uint32_t there = smem_u32(&fac_full[chunk % C::FAC]), there_phase = (chunk / C::FAC) & 1u;
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            if (((told >> h) & 1u) != 0) continue;
            const uint32_t full = smem_u32(&acc_full[2 * (chunk & 1) + h]), phase = (chunk >> 1) & 1u;
            alive = __all_sync(0xFFFFFFFFu, alive && mbar_wait3_tight(full, full, phase, there, there_phase, abort_addr, limit));
            if (!alive) {
              report_timeout(abort_flag, 34);
              told |= 1u << h;
            }
            (void)named_barrier_or(3 + h, 160, !alive);
          }
        }
      }
    }
  } else {
    // ------------------------------ fold and epilogue ------------------------------
    setmaxnreg_inc<C::REGS_FOLD>();
    // (What lives across the chunks beside the sums and the pieces is kept small: registers that spill cost a tenth and more,
    // as hardly any L1 is left beside the shared memory.)
    const int half = (warp - 4) >> 2;
    const uint32_t t_lane = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(half * 128);
    const uint32_t bar_gone = mapa_u32(smem_u32(acc_empty + half), 0);
    const uint32_t fac_row = smem_u32(row_fac) + (uint32_t)((B_ROWS ? 0 : half * 128) + (warp & 3) * 32 + lane) * 4u;
    const uint32_t fac_half = smem_u32(fac) + (uint32_t)half * 512u;    // this half's column factors of a slot
    uint32_t chunk = 0;
    for (uint32_t tile = pair; tile < lists.n_tiles(); tile += gridDim.x >> 1) {
      int chunks = f8_tile(args, lists, tile).chunks;
      float2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = make_float2(0.0f, 0.0f);
      bool alive = true;
      for (; chunks > 0; --chunks, ++chunk) {
        alive = !named_barrier_or(3 + half, 160, false);      // the chunk's accumulator and factors are there
        if (!alive) break;
        tc_fence_after();
        uint32_t r[2][32];
        const uint32_t buf = chunk & 1u, t_acc = t_lane + buf * C::BN;
        tc_ld32(t_acc, r[0]);
        tc_ld32(t_acc + 32, r[1]);
        const float f = ld_shared_f32(fac_row + (chunk % C::ROW_FAC) * 1024u);
        const uint32_t fcol = fac_half + (chunk % C::FAC) * (C::BN * 4);
        auto fold = [&](int p) { f8_fold<B_ROWS>(acc + 16 * p, r[p & 1], f, fcol + 128u * p); };
        tc_wait_ld();
        tc_landed32(r[0]);
        tc_landed32(r[1]);
        fold(0);
        tc_ld32(t_acc + 64, r[0]);
        fold(1);
        tc_ld32(t_acc + 96, r[1]);
        tc_wait_ld();
        tc_fence_before();
        mbar_arrive_cluster_one(bar_gone + 16 * buf);
        tc_landed32(r[0]);
        tc_landed32(r[1]);
        fold(2);
        fold(3);
      }
      if (!alive) break;
      // ---- epilogue: 32 rows x 128 columns, in units of 128 bytes a row ----
      const F8Tile t = f8_tile(args, lists, tile);
      const int thread = (int)thread_here(), lane = thread & 31, warp = thread >> 5, half = (warp - 4) >> 2;
      uint8_t* const epi_warp = epi + (warp - 4) * 8192;
      const uint32_t my_row = smem_u32(epi_warp) + (uint32_t)lane * 128u, sw = (uint32_t)(lane & 7);
      const int e_row = t.row0 + (int)cluster_ctarank() * BM + (warp & 3) * 32, e_rows = t.row_end - e_row, e_col = t.nb * C::BN + half * 128, e_batch = t.batch;
      // (after a failure the wait warp tells at the next chunk)
      if (e_rows <= 0 || e_col >= args.N || __any_sync(0xFFFFFFFFu, *abort_flag != 0)) continue;
      constexpr int ESZ = OUT_BF16 ? 2 : 4, COLS = 128 / ESZ, UNITS = 128 / COLS;
      const bool whole = args.mode != 1 || e_rows >= 32;  // (a copy clips at M, not at the run's end)
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        if ((u & 1) == 0) {                               // both buffers have been read
          if (lane == 0) bulk_wait_read<0>();
          __syncwarp();
        }
        const uint32_t at = my_row + (u & 1) * 4096u;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (OUT_BF16) {
              const float2 v = acc[u * (COLS / 2) + q * 4 + e];
              o[e] = pack_bf16_rn(v.x, v.y);
            } else {
              const float2 v = acc[u * (COLS / 2) + q * 2 + (e >> 1)];
              // (into registers of its own, by an addition of -0: stored from where they are, the sums would have to lie in
              // fours, and some would spill in the loop above)
              asm volatile("add.f32 %0, %1, 0f80000000;" : "=r"(o[e]) : "f"((e & 1) ? v.y : v.x));
            }
          }
          st_shared_v4(at + ((((uint32_t)q) ^ sw) << 4), o[0], o[1], o[2], o[3]);
        }
        if ((u & 1) == 0) continue;
        const int col = e_col + (u - 1) * COLS;           // of the two units
        if (whole) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (col < args.N) tma_store_3d(epi_warp, &tmap_d, col, e_row, e_batch);
            if (col + COLS < args.N) tma_store_3d(epi_warp + 4096, &tmap_d, col + COLS, e_row, e_batch);
            bulk_commit();
          }
        } else {
          __syncwarp();
          const int q = lane & 7;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int cq = col + w * COLS + q * (16 / ESZ);
            if (cq < args.N)
              for (int i = lane >> 3; i < e_rows; i += 4)
                *reinterpret_cast<uint4*>(static_cast<char*>(args.d) + ((int64_t)(e_row + i) * args.ldd + cq) * ESZ) =
                    *reinterpret_cast<const uint4*>(epi_warp + w * 4096 + i * 128 + ((q ^ (i & 7)) << 4));
          }
          __syncwarp();
        }
      }
    }
    if ((threadIdx.x & 31) == 0) bulk_wait_all();
  }

  // ------------------------------ teardown ------------------------------
  // Neither CTA may leave while its peer can still arrive on its barriers or read its shared memory.
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t to = mapa_u32(smem_u32(const_cast<uint32_t*>(ends) + 1), rank ^ 1u);
    st_cluster_u32(to, ends[0]);
    st_cluster_u32(to + 4, (uint32_t)*abort_flag);
  }
  __syncwarp();
  cluster_sync_all();
  if (((uint32_t)*abort_flag | ends[2]) != 0u) {
    // A role of either CTA gave up (both know): copies and MMAs that are on their way land.  (Where none did, all have been waited for.)
    const uint32_t never_addr = smem_u32(const_cast<int*>(never));
    const uint64_t patience = drain_limit(limit);
    if (warp == 0) {
      if (B_ROWS) drain_ring<C::FAC>(fac_full, ends[0], never_addr, patience);
      if (leader) drain_pair<C::STAGES, C::STAGE_BYTES>(full_bar, ends[0], ends[1], lane, never_addr, patience);
    } else if (warp == 1) {
      if (leader && elect_one()) tc_commit_pair(mma_done);
      __syncwarp();
      (void)mbar_wait_tight(smem_u32(mma_done), 0, never_addr, patience);
    }
    __syncwarp();
    cluster_sync_all();
  }
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}
