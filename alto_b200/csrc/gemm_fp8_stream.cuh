// FP8 products of few rows of A (16, or six an expert, or what two rounds of tiles hold): B, the weights, streams through
// shared memory.
//
//   D[m, n] = sum over chunks c of 128 along K of sa[m, c] * sb[n, c] * sum_{k in c} A[m, k] * B[n, k]
//
// Bound by the reading of B up to eight rows, beyond by the instructions: 1 | 16 | 32 rows past 14336 x 4096 take 14.4 | 19.2 |
// 30.4 us (B alone: 9.0), 1 | 16 | 24 | 32 past 4096 x 4096 6.3 | 7.5 | 8.3 | 9.7, 64 rows over 32 experts of 5760 x 2880 80
// (81 for all of them, some are empty).
// tcgen05 on the same stages, 128 rows of B its M side, takes 17.0 | 18.5 | 21.7 and 8.9 | 10.0 | 12 us: a tile of 128 rows of B
// leaves 36 of 148 SMs idle at 14336 and has to be split along K below that, at 1.5 us a join.
//
// A CTA (one an SM, a contiguous range of tiles of up to 16 NW rows of B) keeps its stages of eight chunks of a tile in flight
// by TMA; a stage's chunks are shared out among eight warps, which take rows of B as the 16-row side of the
// matrix instruction and rows of A as the 8-column side, scale a chunk's products and add them in fp32.  The warps' sums are
// joined through shared memory in their order.  A lane's 16 bytes of a row are four instructions' operands: which of a chunk's
// numbers meet in one instruction does not matter as long as both sides agree, so nothing is shuffled.  Codes go through the
// fp16 instruction, in which every code is exact: the one for 8-bit operands converts both sides on every use.
#pragma once
// (included by gemm_sm100.cu inside namespace altob200, after the kernels it shares helpers with)

struct StreamArgs {
  int64_t M, N, K;
  const float *sa, *sb;
  int64_t sa_row, sa_chunk, sb_row, sb_chunk, sb_expert;
  int sa_shift, sb_shift;
  const int32_t* offs;
  int experts;
  int out_bf16;
  int b_ready;             // B, its scales and `offs` were complete before the launch in front of this one
  void* d;
  int64_t ldd;
  int rows;                // of B a tile, a multiple of 8 up to 16 NW
  int stages;
  uint64_t wait_ns;
};

struct CfgStream {
  static constexpr int THREADS = 288;                     // eight warps of products, one of loads
  static constexpr int MOST_STAGES = 6;
  static constexpr int MAX_UNITS = 1024;                  // 8 J rows of A and their expert
  static constexpr int MOST_SMEM = 232448;
  __host__ __device__ static constexpr int stage_bytes(int rows, int j) { return 8 * (rows + 8 * j) * 128; }
  __host__ __device__ static constexpr int part_bytes(int nw, int j) { return 8 * 8 * j * (16 * nw + 1) * 4; }
  __host__ __device__ static constexpr int beside(int nw, int j, bool units) {
    return part_bytes(nw, j) + (units ? MAX_UNITS * 12 : 0) + 1024 /*align*/ + 256 /*barriers*/;
  }
};

struct StreamUnit {
  int row0, row1, expert;
};

// The units of `size` rows, by one warp; returns their number (the host has made sure that they fit).  Rows behind the last
// expert are a run of expert `experts`.
__device__ __forceinline__ int stream_units(const StreamArgs& q, int size, int lane, StreamUnit* units) {
  int carry_end = 0, carry = 0;
  for (int e0 = 0; e0 <= q.experts; e0 += 32) {
    const int e = e0 + lane;
    int end = e < q.experts ? __ldg(q.offs + e) : (int)q.M;
    end = end < 0 ? 0 : (int64_t)end > q.M ? (int)q.M : end;
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
    const int before = carry + sum - n;
    for (int i = 0; i < n; ++i) units[before + i] = {start + i * size, end, e < q.experts ? e : q.experts};
    carry_end = __shfl_sync(0xFFFFFFFFu, end, 31);
    carry = __shfl_sync(0xFFFFFFFFu, before + n, 31);
  }
  return carry;
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
// A word of codes as two pairs of fp16.
template <bool E5M2>
__device__ __forceinline__ void stream_halves(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E5M2)
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e5m2x2 %0, a;\n\tcvt.rn.f16x2.e5m2x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
  else
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ void stream_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NW, int J, bool E5M2>
__global__ void __launch_bounds__(CfgStream::THREADS, 1) fp8_stream_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const StreamArgs q) {
  using C = CfgStream;
  constexpr int A_BOX = 8 * J * 128, PITCH = 16 * NW + 1;
  const int ROWS = q.rows, STAGE = C::stage_bytes(ROWS, J), BOX = ROWS * 128, A_OFF = 8 * BOX;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* const part = reinterpret_cast<float*>(smem + q.stages * STAGE);               // [8 warps][8 J][PITCH]
  uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + q.stages * STAGE + C::part_bytes(NW, J));
  uint64_t *const full = bars, *const empty = bars + C::MOST_STAGES;
  volatile int* const abort_flag = reinterpret_cast<volatile int*>(bars + 2 * C::MOST_STAGES);
  volatile int *const count = abort_flag + 1, *const never = abort_flag + 2;      // never: an abort flag that nothing raises
  StreamUnit* const units = reinterpret_cast<StreamUnit*>(reinterpret_cast<uint8_t*>(bars) + 256);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < q.stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 8);
    }
    *abort_flag = 0;
    *never = 0;
    *count = (int)((q.M + 8 * J - 1) / (8 * J));      // (units of a matrix need no list)
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const bool early = q.b_ready != 0;        // the loads of B need not wait for what makes A
  if (!early) grid_dependency_wait();
  if (q.offs != nullptr) {
    if (warp == 8) {
      const int n = stream_units(q, 8 * J, lane, units);
      if (lane == 0) *count = n;
    }
    __syncthreads();
  }
  const uint32_t abort_addr = smem_u32(const_cast<int*>(abort_flag));
  const uint64_t limit = q.wait_ns * 2ull;
  const int tiles_n = (int)((q.N + ROWS - 1) / ROWS), chunks = (int)((q.K + 127) / 128);
  // this CTA's tiles, unit after unit
  const int64_t total = (int64_t)*count * tiles_n;
  const int64_t t0 = total * blockIdx.x / gridDim.x;
  int left = (int)(total * (blockIdx.x + 1) / gridDim.x - t0), unit = (int)(t0 / tiles_n), col = (int)(t0 - (int64_t)unit * tiles_n);
  const auto unit_at = [&]() -> StreamUnit {
    if (q.offs != nullptr) return units[unit];
    return {unit * 8 * J, (int)q.M, 0};
  };
  const auto step = [&]() {
    --left;
    if (++col == tiles_n) {
      col = 0;
      ++unit;
    }
  };

  if (warp == 8) {
    // ------------------------------ loads ------------------------------
    const bool elected = elect_one();
    uint32_t s = 0, phase = 1, loaded = 0;
    bool alive = true;
    // which: 1 the stage's rows of B, 2 of A; the barrier is armed with those of B
    const auto load = [&](int which, int y, int m, int c, uint32_t to) {
      const int boxes = chunks - c < 8 ? chunks - c : 8;
      if (elected) {
        uint8_t* const st = smem + to * STAGE;
        if (which & 1) {
          mbar_expect_tx(&full[to], (uint32_t)(boxes * (BOX + A_BOX)));
          for (int i = 0; i < boxes; ++i) tma_load_2d(st + i * BOX, &tmap_b, (c + i) * 128, y, &full[to]);
        }
        if (which & 2)
          for (int i = 0; i < boxes; ++i) tma_load_2d(st + A_OFF + i * A_BOX, &tmap_a, (c + i) * 128, m, &full[to]);
      }
      __syncwarp();
    };
    int skip = 0;                // stages whose rows of B are on their way already
    if (early) {
      const int had_left = left, had_unit = unit, had_col = col;
      for (; left > 0 && skip < q.stages; step())
        if (const int e = unit_at().expert; e != q.experts)
          for (int c = 0; c < chunks && skip < q.stages; c += 8) load(1, (int32_t)((int64_t)e * q.N + col * ROWS), 0, c, (uint32_t)skip++);
      left = had_left;
      unit = had_unit;
      col = had_col;
      grid_dependency_wait();
    }
    for (; left > 0 && alive; step()) {
      const StreamUnit u = unit_at();
      if (u.expert == q.experts) continue;
      const int32_t y = (int32_t)((int64_t)u.expert * q.N + col * ROWS);
      for (int c = 0; c < chunks; c += 8) {
        if ((int)loaded >= q.stages) alive = __all_sync(0xFFFFFFFFu, mbar_wait_tight(smem_u32(&empty[s]), phase, abort_addr, limit));
        if (!alive) break;
        load((int)loaded < skip ? 2 : 3, y, u.row0, c, s);
        ++loaded;
        if (++s == (uint32_t)q.stages) {
          s = 0;
          phase ^= 1u;
        }
      }
    }
    if (!alive) report_timeout(abort_flag, 41);
    // the copies in flight land before the CTA ends, whoever gave up
    const uint32_t n = (uint32_t)q.stages;
    for (uint32_t i = loaded < n ? 0 : loaded - n; i < loaded; ++i)
      (void)mbar_wait_tight(smem_u32(&full[i % n]), (i / n) & 1u, smem_u32(const_cast<int*>(never)), drain_limit(limit));
    return;
  }

  // ------------------------------ products ------------------------------
  if (early) grid_dependency_wait();
  const int g = lane >> 2, t = lane & 3;
  const uint32_t at0 = smem_u32(smem) + (uint32_t)(warp * BOX + g * 128), a0 = smem_u32(smem) + (uint32_t)(A_OFF + warp * A_BOX + g * 128);
  uint32_t s = 0, phase = 0;
  bool alive = true;
  for (; left > 0; step()) {
    const StreamUnit u = unit_at();
    const int n0 = col * ROWS, m0 = u.row0;
    const bool zeros = u.expert == q.experts;
    float acc[NW][J][4];
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[w][j][i] = 0.0f;
    // scales of the chunk, asked for a stage ahead
    float sa[J][2], sw[2 * NW], sa_next[J][2], sw_next[2 * NW];
    const auto request = [&](int c) {
      if (c >= chunks) return;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t ms = m0 + 8 * j + 2 * t + h;
          sa_next[j][h] = ms < u.row1 ? __ldg(q.sa + (ms >> q.sa_shift) * q.sa_row + c * q.sa_chunk) : 0.0f;
        }
#pragma unroll
      for (int i = 0; i < 2 * NW; ++i) {
        const int64_t n = n0 + 8 * i + g < q.N ? n0 + 8 * i + g : q.N - 1;
        sw_next[i] = __ldg(q.sb + (int64_t)u.expert * q.sb_expert + (n >> q.sb_shift) * q.sb_row + c * q.sb_chunk);
      }
    };
    if (!zeros) request(warp);
    for (int c0 = 0; c0 < (zeros ? 0 : chunks); c0 += 8) {
      const bool mine = c0 + warp < chunks;
#pragma unroll
      for (int j = 0; j < J; ++j) sa[j][0] = sa_next[j][0], sa[j][1] = sa_next[j][1];
#pragma unroll
      for (int i = 0; i < 2 * NW; ++i) sw[i] = sw_next[i];
      request(c0 + 8 + warp);
      alive = __all_sync(0xFFFFFFFFu, mbar_wait_tight(smem_u32(&full[s]), phase, abort_addr, limit));
      if (!alive) break;
      if (mine) {
        uint4 bw[2 * NW][2], aw[J][2];
        const uint32_t at = at0 + s * STAGE, at_a = a0 + s * STAGE;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t place = (uint32_t)((t + 4 * h) ^ g) << 4;
#pragma unroll
          for (int i = 0; i < 2 * NW; ++i) bw[i][h] = ld_shared_v4(at + i * 1024u + place);
#pragma unroll
          for (int j = 0; j < J; ++j) aw[j][h] = ld_shared_v4(at_a + j * 1024u + place);
        }
        float p[NW][J][4];
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) p[w][j][i] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t v[NW][4], x[J][2];
#pragma unroll
            for (int w = 0; w < NW; ++w) {
              stream_halves<E5M2>((&bw[2 * w][h].x)[i], v[w][0], v[w][2]);
              stream_halves<E5M2>((&bw[2 * w + 1][h].x)[i], v[w][1], v[w][3]);
            }
#pragma unroll
            for (int j = 0; j < J; ++j) stream_halves<E5M2>((&aw[j][h].x)[i], x[j][0], x[j][1]);
#pragma unroll
            for (int w = 0; w < NW; ++w)
#pragma unroll
              for (int j = 0; j < J; ++j) stream_mma(p[w][j], v[w][0], v[w][1], v[w][2], v[w][3], x[j][0], x[j][1]);
          }
#pragma unroll
        for (int w = 0; w < NW; ++w)
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[w][j][i] = __fmaf_rn(p[w][j][i], __fmul_rn(sw[2 * w + (i >> 1)], sa[j][i & 1]), acc[w][j][i]);
      }
      __syncwarp();
      mbar_arrive_lane0(smem_u32(&empty[s]), lane);
      if (++s == (uint32_t)q.stages) {
        s = 0;
        phase ^= 1u;
      }
    }
    // (every warp comes here, also after a failure, which all of them learn of at the second barrier)
    if (!alive) report_timeout(abort_flag, 42);
    named_barrier_sync(1, 256);           // the sums of the tile before have been read
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          part[(warp * 8 * J + 8 * j + 2 * t + (i & 1)) * PITCH + 16 * w + g + 8 * (i >> 1)] = acc[w][j][i];
    if (named_barrier_or(1, 256, !alive)) break;
    for (int i = threadIdx.x; i < 8 * J * 16 * NW; i += 256) {
      const int m = i / (16 * NW), n = i % (16 * NW);
      if (n >= ROWS || m0 + m >= u.row1 || n0 + n >= q.N) continue;
      float v = part[m * PITCH + n];
#pragma unroll
      for (int w = 1; w < 8; ++w) v += part[(w * 8 * J + m) * PITCH + n];
      const int64_t to = (int64_t)(m0 + m) * q.ldd + n0 + n;
      if (q.out_bf16) static_cast<__nv_bfloat16*>(q.d)[to] = __float2bfloat16_rn(v);
      else static_cast<float*>(q.d)[to] = v;
    }
  }
}
