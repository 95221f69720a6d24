// FP8 GEMM with one fp32 scale for each block of 128 along K, for sm_100a.
//
//   D[m, n] = sum over chunks c of 128 along K of sa[m, c] * sb[n, c] * sum_{k in c} A[m, k] * B[n, k]
//
// The scales are fp32, so they cannot ride on a block-scaled MMA (8-bit scales): the tensor cores sum one chunk at a time
// into tensor memory and CUDA cores add it, times both scales, to the fp32 result in registers.
//
// A cluster of two CTAs owns 256 x 256 of the output (cta_group::2), each CTA 128 rows of it; 384 threads a CTA:
//   warp 0      producer: per chunk (128 bytes of K) this CTA's 128 rows of A and half of B's 256 by TMA
//   warp 1      MMA issuer (leader): four tcgen05.mma of 256 x 256 x 32 into one of two chunk accumulators of 256 columns,
//               which are all of the tensor memory
//   warp 2      waits for the issuer (as in the block-scaled pair kernel)
//   warp 3      nothing once the list of units is made; fills the warpgroup
//   warps 4-11  fold: per tensor-memory lane quarter two warps of 32 rows x 128 columns, the sums in 128 registers a lane.
//               64 columns of a chunk at a time come into registers; the accumulator is given back when the last have.
// Rows of A may belong to experts in runs of any length (mode 1): a unit of 256 rows begins at a run's first row, rows of the
// next run that a tile holds beyond its own are multiplied by the wrong weights and not stored.  In mode 2 the reduced
// dimension is cut into the experts' runs of whole chunks.
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
  static constexpr int STAGES = 5;
  static constexpr int FOLD_WARPS = 8;
  static constexpr int EPI_BYTES = FOLD_WARPS * 4096;      // 32 rows x 128 bytes a warp
  // Ring of B's column factors, one slot a chunk.  A slot is written again when the MMAs of the chunk STAGES before have
  // finished; these began when the chunk two before them had been read out by every fold warp, which reads a chunk out
  // only after it has added the one before.
  static constexpr int FAC = STAGES + 3;
  static constexpr int FAC_BYTES = FAC * BN * 4;
  static constexpr int MAX_UNITS = 4096, MAX_RUNS = 2048;  // of a launch
  static constexpr int LIST_BYTES = MAX_UNITS * 4 + MAX_RUNS * 4;
  static constexpr int NUM_BARS = 2 * STAGES + 4 + FAC;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_BYTES + FAC_BYTES + LIST_BYTES + 1024 /*align*/ + 512 /*barriers*/;
  static_assert(NUM_BARS * 8 + 32 <= 512, "barrier area");
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
__device__ __forceinline__ void mbar_arrive_cluster_lane0(uint32_t cluster_addr, int lane) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.eq.s32 p, %1, 0;\n\t"
      "@p mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n\t}"
      ::"r"(cluster_addr), "r"(lane)
      : "memory");
}
// The 32 values in r have landed (tcgen05.wait::ld came before): nothing that uses them can move above this.
__device__ __forceinline__ void tc_landed32(uint32_t* r) {
#define ALTOB200_RW8(o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
  asm volatile("" : ALTOB200_RW8(0), ALTOB200_RW8(8), ALTOB200_RW8(16), ALTOB200_RW8(24));
#undef ALTOB200_RW8
}

struct F8Tile {
  int row0, row_end;       // of A: the tile's first one, the end of its run
  int nb, expert, batch;
  int chunk0, chunks;      // along K
};

// mode 1: units (expert << 16 | unit of the run) and runs' first rows; mode 2: the runs' first chunks.
struct F8Lists {
  uint32_t *units, *runs;
  int n_units;
};

__device__ __forceinline__ F8Tile f8_tile(const F8Args& a, const F8Lists& l, uint32_t tile) {
  F8Tile t;
  t.batch = 0;
  t.expert = 0;
  t.chunk0 = 0;
  t.chunks = (int)((a.K + 127) >> 7);
  const uint32_t tiles_n = (uint32_t)a.tiles_n;
  const uint32_t units = a.mode == 1 ? (uint32_t)l.n_units : (uint32_t)((a.M + 255) >> 8);
  if (a.mode == 2) {
    const uint32_t per = units * tiles_n;
    t.batch = (int)(tile / per);
    tile -= (uint32_t)t.batch * per;
    t.chunk0 = (int)l.runs[t.batch];
    t.chunks = (int)l.runs[t.batch + 1] - t.chunk0;
  }
  // groups of group_m units swept across all columns, the unit running fastest: a group's rows of A stay in L2
  const uint32_t gm = (uint32_t)a.group_m, per_group = gm * tiles_n;
  const uint32_t g = tile / per_group, in = tile - g * per_group;
  const uint32_t left = units - g * gm, rows = left < gm ? left : gm;
  const uint32_t nb = in / rows, u = g * gm + in - nb * rows;
  t.nb = (int)nb;
  if (a.mode == 1) {
    const uint32_t w = l.units[u];
    t.expert = (int)(w >> 16);
    t.row0 = (int)(l.runs[t.expert] + (w & 0xFFFFu) * 256u);
    t.row_end = (int)l.runs[t.expert + 1];
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
    int end = e < a.experts ? __ldg(a.offs + e) : e == a.experts ? (int)limit : 0;
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
  float* fac = reinterpret_cast<float*>(epi + C::EPI_BYTES);
  uint32_t* units = reinterpret_cast<uint32_t*>(epi + C::EPI_BYTES + C::FAC_BYTES);
  uint32_t* runs = units + C::MAX_UNITS;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi + C::EPI_BYTES + C::FAC_BYTES + C::LIST_BYTES);
  uint64_t* full_bar = bars;                      // leader: operand bytes of both CTAs
  uint64_t* empty_bar = bars + C::STAGES;         // each CTA, by the leader's commit
  uint64_t* acc_full = bars + 2 * C::STAGES;      // each CTA, by the leader's commit [chunk & 1]
  uint64_t* acc_empty = acc_full + 2;             // leader: the fold warps of both CTAs
  uint64_t* fac_full = acc_empty + 2;             // each CTA: bytes of its own factors
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fac_full + C::FAC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* count = tmem_slot + 2;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();        // 0 = leader
  const bool leader = rank == 0;
  const uint32_t pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * C::FOLD_WARPS);
    }
    for (int f = 0; f < C::FAC; ++f) mbar_init(&fac_full[f], 1);
    *abort_flag = 0;
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
  F8Lists lists = {units, runs, 0};
  uint32_t n_tiles = (uint32_t)((args.M + 255) >> 8) * (uint32_t)args.tiles_n;
  if (args.mode != 0) {
    if (warp == 3) {
      const int n = f8_lists(args, lane, units, runs);
      if (lane == 0) *count = (uint32_t)n;
    }
    __syncthreads();
    lists.n_units = (int)*count;
    n_tiles = args.mode == 1 ? (uint32_t)lists.n_units * (uint32_t)args.tiles_n : n_tiles * (uint32_t)args.experts;
  }

  if (warp < 4) {
    setmaxnreg_dec<C::REGS_SMALL>();
    if (warp == 0) {
      // ------------------------------ producer ------------------------------
      const bool elected = elect_one();
      uint32_t s = 0, phase = 1, slot = 0;
      bool alive = true;
      for (uint32_t tile = pair; tile < n_tiles && alive; tile += n_pairs) {
        const F8Tile t = f8_tile(args, lists, tile);
        const int32_t ya = t.row0 + (int32_t)rank * BM;
        const int32_t yb = (int32_t)((args.mode == 1 ? (int64_t)t.expert * args.N : 0) + (int64_t)t.nb * C::BN + (int64_t)rank * (C::BN / 2));
        const int64_t n0 = (int64_t)t.nb * C::BN;
        const uint32_t fac_bytes = (uint32_t)(args.N - n0 < C::BN ? args.N - n0 : C::BN) * 4u;
        for (int c = 0; c < t.chunks; ++c) {
          alive = __all_sync(0xFFFFFFFFu, mbar_wait_tight(smem_u32(&empty_bar[s]), phase, abort_addr, limit));
          if (!alive) break;
          uint8_t* st = smem + s * C::STAGE_BYTES;
          const int32_t kx = (t.chunk0 + c) * 128;
          if (elected) {
            if (leader) mbar_expect_tx(&full_bar[s], 2 * C::STAGE_BYTES);
            const uint32_t full_leader = mapa_u32(smem_u32(&full_bar[s]), 0);
            tma_load_2d_pair(st, &tmap_a, kx, ya, full_leader);
            tma_load_2d_pair(st + C::A_BYTES, &tmap_b, kx, yb, full_leader);
            if (B_ROWS) {
              mbar_expect_tx(&fac_full[slot], fac_bytes);
              bulk_load(fac + slot * C::BN, args.sb + (int64_t)(t.chunk0 + c) * args.sb_chunk + n0, fac_bytes, &fac_full[slot]);
            }
          }
          __syncwarp();
          if (++slot == C::FAC) slot = 0;
          if (++s == C::STAGES) {
            s = 0;
            phase ^= 1u;
          }
        }
      }
      if (!alive) report_timeout(abort_flag, 31);
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
            if (named_barrier_or(1 + s, 64, false)) { alive = false; break; }
            tc_fence_after();
            const int64_t left = args.K - (int64_t)(t.chunk0 + c) * 128;
            const int n_mma = left >= 128 ? 4 : (int)((left + 31) / 32);
            const uint32_t a_lo = ((smem_base + s * C::STAGE_BYTES) >> 4) | 0x10000u, b_lo = a_lo + (C::A_BYTES >> 4);
            if (elected) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (j < n_mma)
                  tc_mma_f8_pair(tmem_base + buf * C::BN, desc_of(DESC_SW128_HI, a_lo + 2 * j), desc_of(DESC_SW128_HI, b_lo + 2 * j), args.idesc, (uint32_t)j);
              tc_commit_pair(&empty_bar[s]);
              tc_commit_pair(&acc_full[buf]);
            }
            __syncwarp();
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
            const bool drained = mbar_wait_tight(smem_u32(&acc_empty[chunk & 1]), ((chunk >> 1) & 1) ^ 1, abort_addr, limit);
            const bool ok = drained && mbar_wait_tight(smem_u32(&full_bar[s]), phase, abort_addr, limit);
            if (named_barrier_or(1 + s, 64, !ok)) {
              alive = false;
              report_timeout(abort_flag, drained ? 33 : 32);
              break;
            }
            if (++s == C::STAGES) {
              s = 0;
              phase ^= 1u;
            }
          }
        }
      }
    }
  } else {
    // ------------------------------ fold and epilogue ------------------------------
    setmaxnreg_inc<C::REGS_FOLD>();
    const int quad = warp & 3, half = (warp - 4) >> 2;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(half * 128);
    uint8_t* const epi_warp = epi + (warp - 4) * 4096;
    const uint32_t my_row = smem_u32(epi_warp) + (uint32_t)lane * 128u, sw = (uint32_t)(lane & 7);
    const uint32_t bar_gone = mapa_u32(smem_u32(acc_empty), 0);
    uint32_t chunk = 0, slot = 0, slot_phase = 0;
    bool alive = true;
    for (uint32_t tile = pair; tile < n_tiles && alive; tile += n_pairs) {
      const F8Tile t = f8_tile(args, lists, tile);
      const int row_base = t.row0 + (int)rank * BM + quad * 32;      // this warp's first row
      const int col0 = t.nb * C::BN + half * 128;
      const float *pa, *pb = nullptr;
      {
        const int64_t row = row_base + lane < args.M ? row_base + lane : args.M - 1;
        pa = args.sa + (row >> args.sa_shift) * args.sa_row + (int64_t)t.chunk0 * args.sa_chunk;
        if (!B_ROWS) {
          const int64_t blocks = (args.N + 127) >> 7, b = (int64_t)t.nb * 2 + half < blocks ? (int64_t)t.nb * 2 + half : blocks - 1;
          pb = args.sb + (t.expert < args.experts ? (int64_t)t.expert * args.sb_expert : 0) + b * args.sb_row + (int64_t)t.chunk0 * args.sb_chunk;
        }
      }
      // scales two chunks ahead
      float fa[2] = {0.0f, 0.0f}, fb[2] = {1.0f, 1.0f};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (i < t.chunks) {
          fa[i] = __ldg(pa + i * args.sa_chunk);
          if (!B_ROWS) fb[i] = __ldg(pb + i * args.sb_chunk);
        }
      float2 acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = make_float2(0.0f, 0.0f);
      for (int c = 0; c < t.chunks; ++c, ++chunk) {
        const uint32_t buf = chunk & 1u;
        alive = mbar_wait_tight(smem_u32(&acc_full[buf]), (chunk >> 1) & 1u, abort_addr, limit);
        if (B_ROWS && alive) alive = mbar_wait_tight(smem_u32(&fac_full[slot]), slot_phase, abort_addr, limit);
        alive = __all_sync(0xFFFFFFFFu, alive);
        if (!alive) {
          report_timeout(abort_flag, 34);
          break;
        }
        tc_fence_after();
        const uint32_t t_acc = t_lane + buf * C::BN;
        uint32_t r[2][32];
        tc_ld32(t_acc, r[0]);
        tc_ld32(t_acc + 32, r[1]);
        const float f = __fmul_rn(fa[0], fb[0]);
        const float2 f2 = make_float2(f, f);
        fa[0] = fa[1];
        fb[0] = fb[1];
        if (c + 2 < t.chunks) {
          fa[1] = __ldg(pa + (int64_t)(c + 2) * args.sa_chunk);
          if (!B_ROWS) fb[1] = __ldg(pb + (int64_t)(c + 2) * args.sb_chunk);
        }
        const uint32_t fcol = smem_u32(fac) + slot * (C::BN * 4) + (uint32_t)half * 512u;
        auto fold = [&](int p) {
          uint32_t* v = r[p & 1];
          if (B_ROWS) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float4 w = ld_shared_f32x4(fcol + (uint32_t)(p * 32 + 4 * j) * 4u);
              const float2 w0 = __fmul2_rn(f2, make_float2(w.x, w.y)), w1 = __fmul2_rn(f2, make_float2(w.z, w.w));
              acc[p * 16 + 2 * j] = __ffma2_rn(make_float2(u2f(v[4 * j]), u2f(v[4 * j + 1])), w0, acc[p * 16 + 2 * j]);
              acc[p * 16 + 2 * j + 1] = __ffma2_rn(make_float2(u2f(v[4 * j + 2]), u2f(v[4 * j + 3])), w1, acc[p * 16 + 2 * j + 1]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[p * 16 + j] = __ffma2_rn(make_float2(u2f(v[2 * j]), u2f(v[2 * j + 1])), f2, acc[p * 16 + j]);
          }
        };
        tc_wait_ld();
        tc_landed32(r[0]);
        tc_landed32(r[1]);
        fold(0);
        tc_ld32(t_acc + 64, r[0]);
        fold(1);
        tc_ld32(t_acc + 96, r[1]);
        tc_wait_ld();
        tc_fence_before();
        mbar_arrive_cluster_lane0(bar_gone + 8 * buf, lane);
        tc_landed32(r[0]);
        tc_landed32(r[1]);
        fold(2);
        fold(3);
        if (++slot == C::FAC) {
          slot = 0;
          slot_phase ^= 1u;
        }
      }
      if (!alive || __any_sync(0xFFFFFFFFu, *abort_flag != 0)) break;
      // ---- epilogue: 32 rows x 128 columns, in units of 128 bytes a row ----
      const int rows = t.row_end - row_base;            // of this warp's, that are the run's own
      if (rows <= 0 || col0 >= args.N) continue;
      constexpr int ESZ = OUT_BF16 ? 2 : 4, COLS = 128 / ESZ;
      const bool whole = args.mode != 1 || rows >= 32;  // (a copy clips at M, not at the run's end)
#pragma unroll
      for (int u = 0; u < 128 / COLS; ++u) {
        if (lane == 0) bulk_wait_read<0>();
        __syncwarp();
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
              o[e] = f2u((e & 1) ? v.y : v.x);
            }
          }
          st_shared_v4(my_row + ((((uint32_t)q) ^ sw) << 4), o[0], o[1], o[2], o[3]);
        }
        const int col = col0 + u * COLS;
        if (whole) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (col < args.N) tma_store_3d(epi_warp, &tmap_d, col, row_base, t.batch);
            bulk_commit();
          }
        } else {
          __syncwarp();
          const int q = lane & 7, cq = col + q * (16 / ESZ);
          if (cq < args.N)
            for (int i = lane >> 3; i < rows; i += 4)
              *reinterpret_cast<uint4*>(static_cast<char*>(args.d) + ((int64_t)(row_base + i) * args.ldd + cq) * ESZ) =
                  *reinterpret_cast<const uint4*>(epi_warp + i * 128 + ((q ^ (i & 7)) << 4));
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
  }

  // ------------------------------ teardown ------------------------------
  // Neither CTA may leave while its peer can still arrive on its barriers or read its shared memory.
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}
