// Products in 8-bit floating point (fp8.cuh) of few rows, where the bytes of W are what counts:
//   C[t, n] = sum_b s[b, t] S[n / 128, b] sum_{k in block b} q[t, k] Q[n, k].
//
// A CTA takes 128 rows of W (the M of a tcgen05.mma), NX rows of A (its N: 16, 32 or 64) and a range of the blocks of K; the CTAs of a
// cluster take the ranges of one tile.  A block's sums are formed in one of NACC accumulators in tensor memory.  Roles by warp:
//   warps 0 .. 4 ADD - 1   add: a thread owns a row of W and 64 columns at most; it adds a finished accumulator, times the row's and the columns' scales
//                          (their products are in shared memory, CHUNK blocks at a time), to its sums
//   the next one           copies: STAGES blocks of W and A in flight.  W does not depend on what the stream ran before, so its first stages are
//                          asked for before that has ended
//   the one behind it      products
//   four more (FUSED)      quantise: up to 16 rows of activations come as they are (float32 or bfloat16); these warps quantise a block of them into
//                          each stage as the copy of W comes in, and leave its scales for the adding warps
// Behind its range every CTA sends its sums, column by column, to the CTA of the cluster that owns the column; that one adds them in the
// order of the ranges and writes them, neighbouring lanes neighbouring outputs.  So a result depends on the sizes alone.
//
// `starts`: W is a stack of matrices and rows starts[e] .. starts[e + 1] of A meet the e-th.  Gated: rows of W alternate, eight gates and the eight
// ups of the same outputs, each with the scales of their own matrix.
//
// What bounds it: W's bytes where there are enough of them, else the way of a block of K: copy, four products and a commit (0.24 us of issue, whatever N
// is and wherever W lies), tensor memory, sums.  Hence K in parts where tiles are few (0.5 to 0.6 us, and 0.07 to 0.26 for each part), two CTAs a
// multiprocessor, so that one's issue hides the other's, and 128 rows of A on the lanes from some 70 rows on (no factors from shared memory, 64 rows of W a
// tile).  Measured, products behind one another in a graph, quantising included: 1 row by 6,144 x 4,096 6.8 us (25 MB), 8 rows' gate and up of 12,288 x 4,096
// 18.4 (5.5 TB/s; a copy reaches 6.45), 64 by 5,120 x 17,408 18.2 with given rows (4.9 TB/s), 128 by 6,144 x 4,096 11.1, 256 by 4,096 x 4,096 10.9.
//
// Every wait on a barrier gives up after a bounded number of polls and leaves a code in `*status`, as in gemm_tc.cu; the allocation of tensor memory waits for
// CTAs that end whatever this one does (see tmem_alloc).
#pragma once
#include "product_fp8.cuh"

namespace few {

constexpr int LANES = 128, BK = F8_BLOCK, LANE_BYTES = LANES * BK;
enum { ST_PRODUCER_TIMEOUT = 34, ST_MMA_TIMEOUT = 35, ST_ADDER_TIMEOUT = 36, ST_QUANTISER_TIMEOUT = 37 };

constexpr int MOST_SPLIT = 8;
constexpr int MOST_TILES_N = 65535;                      // a product's tiles along W's rows are the grid's second axis
// columns that a CTA of `split` owns, `unit` at a time, and the most that ranges and columns owned come to
constexpr int columns_owned(int columns, int unit, int split) { return (columns / unit + split - 1) / split * unit; }
constexpr int most_sent(int columns, int unit) {
  int most = 0;
  for (int s = 1; s <= MOST_SPLIT; ++s)
    if (columns_owned(columns, unit, s) * s > most) most = columns_owned(columns, unit, s) * s;
  return most;
}

// LANES_A: the tile the other way round, 128 rows of A on the lanes of tensor memory and NX rows of W as its columns.
// Two CTAs a multiprocessor; three with experts' rows in sixteens and half the ring, since an expert's tiles are many and short (64 tokens of 6 choices among 64
// experts of 768 between 2,048: 82 us against 88, weights from DRAM).
template <int NX, bool LANES_A, bool FUSED, bool GROUPED> struct Shape {
  static constexpr bool MORE = GROUPED && !FUSED && NX == 16;
  static constexpr int ADD = NX >= 64 ? 2 : 1;           // groups of four adding warps
  static constexpr int COLS = NX / ADD;
  static constexpr int STAGES = MORE ? 3 : NX == 16 ? 6 : NX == 32 ? 5 : 4;
  static constexpr int NACC = MORE ? 3 : 4;                       // at most STAGES: a stage's barrier says both that its operands and that its sums are done
  static constexpr int CHUNK = NX <= 32 ? 16 : 8;        // blocks whose scales are in shared memory at a time
  static constexpr int PITCH = LANES_A ? LANES + 1 : LANES;                           // of the columns sent: read along rows, or (LANES_A) along columns
  static constexpr int STAGE_BYTES = LANES * BK + NX * BK;
  static constexpr int RING = STAGES * STAGE_BYTES, SENT = most_sent(NX, LANES_A ? 16 : 4) / 4 * PITCH * 16;     // SENT lies where the ring was
  static constexpr int FACTORS = LANES_A ? 0 : 2 * CHUNK * NX * 4;
  static constexpr int SMEM = RING + FACTORS + 512 + 1024;                            // + barriers, + the swizzle's alignment
  static constexpr int THREADS = (4 * ADD + 2 + (FUSED ? 4 : 0)) * 32, PER_SM = MORE ? 3 : 2;
  static constexpr int TMEM = 4 * NX;
  static constexpr int ROWS_A = LANES_A ? LANES : NX, ROWS_W = LANES_A ? NX : LANES;
  static_assert(!FUSED || (CHUNK > STAGES + NACC && NX == 16), "a block's scales stay until its sums are added");
  static_assert((2 * STAGES + NACC + CHUNK) * 8 + (1 + 3 + MOST_INLINE) * 4 <= 512, "barriers and what a tile is found with");
  static_assert(NACC <= STAGES, "an adder must have seen a stage's barrier before its next products are issued");
  static_assert(SENT <= RING && PER_SM * (SMEM + 1024) <= 228 * 1024 && PER_SM * TMEM <= 512, "what a multiprocessor holds");
};

struct Few : Product {
  int nb, split, tiles_n;                                // nb: blocks of W's rows that have a scale
};

template <bool ACC>
__device__ __forceinline__ void umma_f8(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  constexpr uint32_t HIGH = (1024 >> 4) | (1u << 14) | (2u << 29);
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}\n"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(HIGH), "n"(ACC ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// Columns of this thread's lane: asked for, and waited for (the registers pass through the wait, so that nothing that reads them moves in front).
__device__ __forceinline__ void ask_columns(uint32_t from, uint32_t (&x)[1][16]) { tmem_ld16(from, x[0]); }
__device__ __forceinline__ void ask_columns(uint32_t from, uint32_t (&x)[1][32]) { tmem_ld32(from, x[0]); }
__device__ __forceinline__ void ask_columns(uint32_t from, uint32_t (&x)[2][32]) {
  tmem_ld32(from, x[0]);
  tmem_ld32(from + 32, x[1]);
}
__device__ __forceinline__ void got_columns(uint32_t (&x)[1][16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" : F8_RW8(x[0], 0), F8_RW8(x[0], 8) : : "memory");
}
__device__ __forceinline__ void got_columns(uint32_t (&x)[1][32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" : F8_RW8(x[0], 0), F8_RW8(x[0], 8), F8_RW8(x[0], 16), F8_RW8(x[0], 24) : : "memory");
}
__device__ __forceinline__ void got_columns(uint32_t (&x)[2][32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" : F8_RW8(x[0], 0), F8_RW8(x[0], 8), F8_RW8(x[0], 16), F8_RW8(x[0], 24) : : "memory");
  asm volatile("" : F8_RW8(x[1], 0), F8_RW8(x[1], 8), F8_RW8(x[1], 16), F8_RW8(x[1], 24));
}

template <int NX, bool LANES_A, int EPI, bool GROUPED, bool FUSED>
__global__ void __launch_bounds__(Shape<NX, LANES_A, FUSED, GROUPED>::THREADS, Shape<NX, LANES_A, FUSED, GROUPED>::PER_SM)
gemm_fp8_few_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ Few p) {
  using S = Shape<NX, LANES_A, FUSED, GROUPED>;
  constexpr bool GATED = EPI == EPI_GATED_F32;
  constexpr int ADDERS = 4 * S::ADD, CHUNK = S::CHUNK, PIECE = S::COLS < 32 ? S::COLS : 32, PIECES = S::COLS / PIECE;
  constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(NX >> 3) << 17) | ((uint32_t)(LANES >> 4) << 24);      // accumulator float, operands e4m3, K-major
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float4 *sent = reinterpret_cast<float4 *>(smem);                        // [range][four columns owned][row], behind the loop
  float *factors = reinterpret_cast<float *>(smem + S::RING);             // [gate, up][block of the chunk][column]
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::RING + S::FACTORS);
  const uint32_t full0 = smem_addr(bars), done0 = full0 + 8 * S::STAGES, sum_empty0 = done0 + 8 * S::STAGES, scaled0 = sum_empty0 + 8 * S::NACC;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * S::STAGES + S::NACC + (FUSED ? CHUNK : 0));
  int *found = reinterpret_cast<int *>(tmem_slot + 1), *pair_of = found + 3;              // pair_of: with p.idx, the pair of every row
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // Tiles of other rows of A, which read the same W, are neighbours.  Of experts, whose tiles along M are fewer than the grid's, those that are none come last.
  const int rank = (int)(blockIdx.x % p.split), tile = (int)(blockIdx.x / p.split);
  const int tile_m = GROUPED ? tile / p.tiles_n : tile, n0 = (GROUPED ? tile - tile_m * p.tiles_n : (int)blockIdx.y) * S::ROWS_W;
  const int per = (p.blocks + p.split - 1) / p.split, kb0 = rank * per, nkb = max(0, min(p.blocks, kb0 + per) - kb0);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(full0 + 8 * s, FUSED ? 5 : 1);           // the copies' bytes; the quantising warps
      mbar_init(done0 + 8 * s, 1);
    }
    for (int b = 0; b < S::NACC; ++b) mbar_init(sum_empty0 + 8 * b, ADDERS);
    if (FUSED)
      for (int b = 0; b < CHUNK; ++b) mbar_init(scaled0 + 8 * b, 4);
    mbar_init_fence();
  }
  // Tensor memory under the wait for the kernel in front; but many tiles of experts, a part of them none, take theirs once they know (64 tokens of 6 choices:
  // 67.5 us against 70.4; one token, which quantises on the way: 17.2 against 16.0).
  constexpr bool EARLY = !GROUPED || FUSED;
  auto take_tensor_memory = [&] {
    tmem_alloc(smem_addr(tmem_slot), S::TMEM);
    pdl_launch();                                        // only now: see tmem_alloc
  };
  if (EARLY && warp == ADDERS + 1) take_tensor_memory();
  tc_fence_before();
  int e = 0, m0 = tile_m * S::ROWS_A, end = p.M;
  if (GROUPED) {
    pdl_wait();
    if (FUSED && p.idx) {
      // Few pairs: every CTA sorts them for itself, a pair a lane (a launch less: one token's four choices 32.5 -> 29.1 us).  A lane counts the pairs of
      // smaller experts, and those of its own in front of it; a tile begins at every ROWS_A-th row of an expert.
      if (warp == 0) {
        const int n = p.M, x = lane < n ? p.idx[lane] : -1, own = x >= 0 && x < p.n_experts ? x : p.n_experts;
        int first = 0, count = 0, row = 0, before = 0;
        for (int i = 0; i < n; ++i) {
          const int y = __shfl_sync(0xffffffffu, own, i);
          first += y < own, count += y == own, row += y == own && i < lane;
        }
        const bool begins = lane < n && own < p.n_experts && row % S::ROWS_A == 0;
        const uint32_t all = __ballot_sync(0xffffffffu, begins);
        row += first;
        for (int i = 0; i < n; ++i) {
          const int y = __shfl_sync(0xffffffffu, row, i);
          before += (all >> i & 1) && y < row;
        }
        const bool hit = begins && before == tile_m;
        if (hit) found[0] = own, found[1] = row, found[2] = first + count;
        if (!__any_sync(0xffffffffu, hit) && lane == 0) found[0] = -1;
        if (lane < n) {
          pair_of[row] = lane;
          if (p.pair_row && blockIdx.x == 0) p.pair_row[lane] = own < p.n_experts ? row : -1;
        }
      }
    } else if (warp == 0) {                              // which expert's which rows: a lane counts the tiles of `each` neighbouring experts
      const int each = (p.n_experts + 31) / 32, e0 = min(lane * each, p.n_experts), e1 = min(e0 + each, p.n_experts);
      int own = 0, first = p.starts[e0];
#pragma unroll 4
      for (int x = e0; x < e1; ++x) {
        const int behind = p.starts[x + 1];
        own += (behind - first + S::ROWS_A - 1) / S::ROWS_A;
        first = behind;
      }
      int sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const bool hit = sum > tile_m && sum - own <= tile_m;
      if (hit) {                                         // (one lane at most; its experts' starts are in the L1 now)
        int left = tile_m - (sum - own);
        for (int x = e0; x < e1; ++x) {
          const int row = p.starts[x], behind = p.starts[x + 1], tiles = (behind - row + S::ROWS_A - 1) / S::ROWS_A;
          if (left < tiles) {
            found[0] = x, found[1] = row + left * S::ROWS_A, found[2] = behind;
            break;
          }
          left -= tiles;
        }
      }
      if (!__any_sync(0xffffffffu, hit) && lane == 0) found[0] = -1;
    }
    __syncwarp();
  }
  __syncthreads();
  tc_fence_after();
  if (GROUPED) {
    e = found[0], m0 = found[1], end = found[2];
    if (e < 0) {                                         // (the whole cluster: its CTAs have one tile)
      if (EARLY && warp == ADDERS + 1) tmem_dealloc(*tmem_slot, S::TMEM);
      return;
    }
  }
  if (!EARLY) {
    if (warp == ADDERS + 1) take_tensor_memory();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }
  const uint32_t tmem = *tmem_slot;

  if (warp == ADDERS) {
    if (PRODUCER_RUNS) {
      const int row_w = e * p.N + n0, at_w = LANES_A ? LANE_BYTES : 0, at_a = LANE_BYTES - at_w;
      const int ahead = min(nkb, S::STAGES);
      if (elect_one()) {
        for (int i = 0; i < ahead; ++i) {
          mbar_expect_tx(full0 + 8 * i, FUSED ? LANE_BYTES : S::STAGE_BYTES);
          tma_load_2d(smem_addr(smem + i * S::STAGE_BYTES) + at_w, &map_w, (kb0 + i) * BK, row_w, full0 + 8 * i);
        }
        if (!GROUPED && !FUSED) pdl_wait();
        for (int i = 0; i < ahead && !FUSED; ++i) tma_load_2d(smem_addr(smem + i * S::STAGE_BYTES) + at_a, &map_a, (kb0 + i) * BK, m0, full0 + 8 * i);
      }
      __syncwarp();
      if (!GROUPED && FUSED) pdl_wait();
      for (int i = ahead; i < nkb; ++i) {
        const int s = i % S::STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(done0 + 8 * s, (i / S::STAGES - 1) & 1))) {
          if (lane == 0) atomicExch(p.status, ST_PRODUCER_TIMEOUT);
          break;
        }
        const uint32_t to = smem_addr(smem + s * S::STAGE_BYTES);
        if (elect_one()) {
          mbar_expect_tx(full0 + 8 * s, FUSED ? LANE_BYTES : S::STAGE_BYTES);
          tma_load_2d(to + at_w, &map_w, (kb0 + i) * BK, row_w, full0 + 8 * s);
          if (!FUSED) tma_load_2d(to + at_a, &map_a, (kb0 + i) * BK, m0, full0 + 8 * s);
        }
        __syncwarp();
      }
    }
    __syncwarp();
  } else if (warp == ADDERS + 1) {
    if (!GROUPED) pdl_wait();                            // (the kernel in front may take longer than a wait is bounded by)
    for (int i = 0; i < nkb; ++i) {
      const int s = i % S::STAGES, h = i % S::NACC;
      const bool ok = mbar_wait(full0 + 8 * s, (i / S::STAGES) & 1) && (i < S::NACC || mbar_wait(sum_empty0 + 8 * h, (i / S::NACC - 1) & 1));
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) atomicExch(p.status, ST_MMA_TIMEOUT);
        break;
      }
      tc_fence_after();
      const uint32_t lo = ((smem_addr(smem + s * S::STAGE_BYTES) & 0x3FFFF) >> 4) | 1u << 16;
      const uint32_t to = tmem + h * NX;
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (k == 0) umma_f8<false>(to, lo, lo + LANE_BYTES / 16, IDESC);
          else umma_f8<true>(to, lo + 2 * k, lo + LANE_BYTES / 16 + 2 * k, IDESC);
        }
        umma_commit(done0 + 8 * s);
      }
      __syncwarp();
    }
  } else if (FUSED && warp > ADDERS + 1) {
    if (!GROUPED) pdl_wait();
    // eight lanes a row, sixteen values each; AHEAD blocks are asked for before the first one is used
    const int r = (threadIdx.x - (ADDERS + 2) * 32) / 8, part = threadIdx.x % 8;
    const bool live = m0 + r < end;
    const int source = !live ? 0 : GROUPED && p.idx && p.gather ? pair_of[m0 + r] / p.top : p.row_pair ? p.row_pair[m0 + r] / p.top : m0 + r;
    const long long from = source * p.x_stride;
    const int n_block = min((GATED ? n0 / 2 : n0) / F8_BLOCK, p.nb - 1);
    const float *sw = p.sw + ((long long)e * (GATED ? 2 : 1) * p.nb + n_block) * p.blocks + kb0;
    bool ok = true;
    auto walk = [&](auto one) {
      using T = decltype(one);
      constexpr int PER16 = 16 / sizeof(T), LOADS = 16 / PER16, AHEAD = 8 / LOADS;
      uint4 raw[AHEAD][LOADS];
      float next_w[AHEAD], next_up[AHEAD];
      auto ask = [&](int u, int i) {
        if (i >= nkb) return;
        const int k = (kb0 + i) * BK + 16 * part;        // K is a multiple of 8
#pragma unroll
        for (int j = 0; j < LOADS; ++j)
          raw[u][j] = live && k + PER16 * j < p.K ? *reinterpret_cast<const uint4 *>(static_cast<const T *>(p.x) + from + k + PER16 * j) : make_uint4(0, 0, 0, 0);
        next_w[u] = sw[i];
        next_up[u] = GATED ? sw[(long long)p.nb * p.blocks + i] : 0.f;
      };
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) ask(u, u);
      for (int i0 = 0; i0 < nkb && ok; i0 += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int i = i0 + u, s = i % S::STAGES;
          if (i >= nkb || !ok) break;
          float v[16], most = 0.f;
#pragma unroll
          for (int j = 0; j < LOADS; ++j) {
            const uint32_t w[4] = {raw[u][j].x, raw[u][j].y, raw[u][j].z, raw[u][j].w};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if constexpr (sizeof(T) == 4) v[4 * j + x] = __uint_as_float(w[x]);
              else v[8 * j + 2 * x] = __uint_as_float(w[x] << 16), v[8 * j + 2 * x + 1] = __uint_as_float(w[x] & 0xffff0000u);
            }
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) most = max_nan(most, fabsf(v[j]));
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
          const BlockScale b = block_scale(most);
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = pack_e4m3(v[4 * j] * b.inverse, v[4 * j + 1] * b.inverse, v[4 * j + 2] * b.inverse, v[4 * j + 3] * b.inverse);
          const float f = b.scale * next_w[u], f_up = b.scale * next_up[u];
          ask(u, i + AHEAD);
          if (i >= S::STAGES) ok = __all_sync(0xffffffffu, mbar_wait(done0 + 8 * s, (i / S::STAGES - 1) & 1));
          if (!ok) {
            if (lane == 0) atomicExch(p.status, ST_QUANTISER_TIMEOUT);
            break;
          }
          *reinterpret_cast<uint4 *>(smem + s * S::STAGE_BYTES + LANE_BYTES + r * 128 + ((part ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          if (part == 0) {
            factors[i % CHUNK * NX + r] = f;
            if (GATED) factors[CHUNK * NX + i % CHUNK * NX + r] = f_up;
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(full0 + 8 * s);
            mbar_arrive(scaled0 + 8 * (i % CHUNK));
          }
        }
      }
    };
    if (p.x_f32) walk(0.f);
    else walk(bf16());
    __syncwarp();
  }
  // columns that a CTA writes (rows of A, or outputs), four at a time, or gates and ups of eight; the last CTAs maybe fewer, or none
  constexpr int UNIT = LANES_A && GATED ? 16 : 4;
  const int own = columns_owned(NX, UNIT, p.split);
  if (warp < ADDERS) {
    if (!GROUPED) pdl_wait();
    const int row = 32 * (warp % 4) + lane, col0 = S::COLS * (warp / 4);
    const uint32_t from0 = tmem + ((uint32_t)(32 * (warp % 4)) << 16) + col0;
    const int n_block = min((GATED ? n0 / 2 : n0) / F8_BLOCK, p.nb - 1);
    const float *sw = p.sw + ((long long)e * (GATED ? 2 : 1) * p.nb + n_block) * p.blocks + kb0;
    const float *mine = factors + (GATED && (row & 8) ? CHUNK * NX : 0) + col0;
    float sum[S::COLS];
#pragma unroll
    for (int j = 0; j < S::COLS; ++j) sum[j] = 0.f;
    constexpr int PER = FUSED ? 1 : LANES_A ? 4 : CHUNK * NX / (ADDERS * 32);        // LANES_A: the scales of the next four blocks
    float next_a[PER], next_w[PER], next_up[PER];
    auto ask = [&](int first) {                          // the scales of a chunk that the thread brings, all at once
#pragma unroll
      for (int x = 0; x < PER; ++x) {
        const int at = threadIdx.x + x * ADDERS * 32, b = min(first + (LANES_A ? x : at / NX), nkb - 1), t = m0 + (LANES_A ? row : at % NX);
        next_a[x] = t < p.M ? p.sa[(kb0 + b) * p.lds + t] : 0.f;
        next_w[x] = sw[b];
        next_up[x] = GATED ? sw[(long long)p.nb * p.blocks + b] : 0.f;
      }
    };
    if (nkb > 0 && !FUSED) ask(0);
    float four[PER] = {}, four_up[PER] = {};
    bool ok = true;                                      // once a wait gave up nothing is waited for any more (the warps still meet at their barriers)
    for (int i = 0; i < nkb; ++i) {
      const int h = i % S::NACC;
      float f_row = 0.f, f_up = 0.f;
      if (LANES_A) {                                     // the scales of the thread's row and of the tile's columns
        if (i % PER == 0) {
#pragma unroll
          for (int x = 0; x < PER; ++x) four[x] = next_a[x] * next_w[x], four_up[x] = next_a[x] * next_up[x];
          if (i + PER < nkb) ask(i + PER);
        }
        f_row = four[0], f_up = four_up[0];
#pragma unroll
        for (int x = 1; x < PER; ++x) four[x - 1] = four[x], four_up[x - 1] = four_up[x];
      } else if (!FUSED && i % CHUNK == 0) {             // this chunk's scales are in registers: to shared memory, and the next chunk's asked for
        if (i) asm volatile("bar.sync 1, %0;\n" ::"n"(ADDERS * 32) : "memory");
#pragma unroll
        for (int x = 0; x < PER; ++x) {
          factors[threadIdx.x + x * ADDERS * 32] = next_a[x] * next_w[x];
          if (GATED) factors[CHUNK * NX + threadIdx.x + x * ADDERS * 32] = next_a[x] * next_up[x];
        }
        asm volatile("bar.sync 1, %0;\n" ::"n"(ADDERS * 32) : "memory");
        if (i + CHUNK < nkb) ask(i + CHUNK);
      }
      if (ok) {
        ok = __all_sync(0xffffffffu, (!FUSED || mbar_wait(scaled0 + 8 * (i % CHUNK), (i / CHUNK) & 1)) && mbar_wait(done0 + 8 * (i % S::STAGES), (i / S::STAGES) & 1));
        if (!ok && lane == 0) atomicExch(p.status, ST_ADDER_TIMEOUT);
      }
      if (!ok) continue;
      tc_fence_after();
      const float *f = mine + i % CHUNK * NX;
      uint32_t x[PIECES][PIECE];
      ask_columns(from0 + h * NX, x);
      got_columns(x);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sum_empty0 + 8 * h);
#pragma unroll
      for (int c = 0; c < S::COLS; c += 4) {
        const uint32_t *v = &x[c / PIECE][c % PIECE];
        const float g = GATED && (c & 8) ? f_up : f_row;
        const float4 s = LANES_A ? make_float4(g, g, g, g) : *reinterpret_cast<const float4 *>(f + c);
        const float2 u0 = fma2(make_float2(__uint_as_float(v[0]), __uint_as_float(v[1])), make_float2(s.x, s.y), make_float2(sum[c], sum[c + 1]));
        const float2 u1 = fma2(make_float2(__uint_as_float(v[2]), __uint_as_float(v[3])), make_float2(s.z, s.w), make_float2(sum[c + 2], sum[c + 3]));
        sum[c] = u0.x, sum[c + 1] = u0.y, sum[c + 2] = u1.x, sum[c + 3] = u1.y;
      }
    }
    // Four columns at a time go to the CTA that owns them, as range `rank`'s part, to where that one's ring was: once the sums of all are complete nobody's
    // products read a ring any more.
    if (p.split > 1) cluster_sync_all();
    if (p.split == 1) {
#pragma unroll
      for (int j = 0; j < S::COLS; j += 4)
        sent[(col0 + j) / 4 * S::PITCH + row] = make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]);
    } else {
      const uint32_t base = smem_addr(sent);
      int to = col0 / own, left = own - col0 % own;      // the owner of the columns at hand, and how many of its own are still to come
#pragma unroll
      for (int j = 0; j < S::COLS; j += 4) {
        const uint32_t at = base + ((rank * own + own - left) / 4 * S::PITCH + row) * 16;
        st_cluster(map_to_cta(at, (uint32_t)to), make_float4(sum[j], sum[j + 1], sum[j + 2], sum[j + 3]));
        left -= 4;
        if (left == 0) ++to, left = own;
      }
    }
  } else if (p.split > 1) {
    cluster_sync_all();
  }
  tc_fence_before();
  if (p.split == 1) __syncthreads();
  else cluster_sync_all();
  if (warp == ADDERS + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM);
  }
  // four columns from the `c`-th owned on, of lane r: the ranges' parts in their order
  auto whole = [&](int c, int r) {
    float4 v = sent[c / 4 * S::PITCH + r];
#pragma unroll
    for (int s = 1; s < MOST_SPLIT; ++s) {
      if (s >= p.split) break;
      const float4 x = sent[(s * own + c) / 4 * S::PITCH + r];
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
    }
    return v;
  };
  if (warp < ADDERS && LANES_A) {                        // neighbouring lanes neighbouring fours of a row's outputs
    constexpr int STEP = GATED ? 8 : 4;                  // columns behind four outputs
    const int columns = min(own, NX - rank * own), fours = max(1, columns / STEP), n_out = GATED ? p.N / 2 : p.N;
    const int first = (n0 + rank * own) / (GATED ? 2 : 1);
    const bool vector = p.ldo % 4 == 0 && ((uintptr_t)p.out & (EPI == EPI_BF16 ? 7 : 15)) == 0;
    for (int x = threadIdx.x; columns > 0 && x < LANES * fours; x += ADDERS * 32) {
      const int r = x / fours, q = x - r * fours, n = first + 4 * q;
      if (m0 + r >= end) break;
      if (n >= n_out) continue;
      const long long at = (long long)(m0 + r) * p.ldo + n;
      float *const to = static_cast<float *>(p.out) + at;
      const bool all = vector && n + 4 <= n_out;
      float4 old = make_float4(0.f, 0.f, 0.f, 0.f);
      if (EPI == EPI_ADD_F32 && all) old = *reinterpret_cast<const float4 *>(to);
      float4 v = whole(GATED ? (q >> 1) * 16 + (q & 1) * 4 : 4 * q, r);
      if (GATED) {
        const float4 u = whole((q >> 1) * 16 + (q & 1) * 4 + 8, r);
        v = make_float4(glu_value(v.x, u.x, p.form), glu_value(v.y, u.y, p.form), glu_value(v.z, u.z, p.form), glu_value(v.w, u.w, p.form));
      }
      if (all) {
        if (EPI == EPI_BF16) {
          const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
          *reinterpret_cast<uint2 *>(static_cast<bf16 *>(p.out) + at) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
        } else {
          *reinterpret_cast<float4 *>(to) = EPI == EPI_ADD_F32 ? make_float4(old.x + v.x, old.y + v.y, old.z + v.z, old.w + v.w) : v;
        }
      } else {
        const float vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (n + i >= n_out) break;
          if (EPI == EPI_BF16) static_cast<bf16 *>(p.out)[at + i] = __float2bfloat16_rn(vs[i]);
          else to[i] = EPI == EPI_ADD_F32 ? to[i] + vs[i] : vs[i];
        }
      }
    }
  } else if (warp < ADDERS) {                            // neighbouring lanes neighbouring outputs, four rows at a time
    const int t0 = m0 + rank * own, rows = min(min(own, NX - rank * own), end - t0);
    constexpr int OUTS = GATED ? LANES / 2 : LANES;      // outputs of a row of A
    const int n = (GATED ? n0 / 2 : n0) + threadIdx.x % OUTS, n_out = GATED ? p.N / 2 : p.N;
    if (n < n_out) {
      const int l = threadIdx.x % OUTS, r0 = GATED ? (l >> 3) * 16 + (l & 7) : l;
      for (int c = threadIdx.x / OUTS * 4; c < rows; c += ADDERS * 32 / OUTS * 4) {
        const long long at = (long long)(t0 + c) * p.ldo + n;
        float *const add = static_cast<float *>(p.out) + at;
        float4 old = make_float4(0.f, 0.f, 0.f, 0.f);
        if (EPI == EPI_ADD_F32)
          old = make_float4(add[0], c + 1 < rows ? add[p.ldo] : 0.f, c + 2 < rows ? add[2 * p.ldo] : 0.f, c + 3 < rows ? add[3 * p.ldo] : 0.f);
        const float4 v = whole(c, r0), u = GATED ? whole(c, r0 + 8) : v;
        const float vs[4] = {v.x, v.y, v.z, v.w}, us[4] = {u.x, u.y, u.z, u.w}, olds[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (c + i >= rows) break;
          if (GATED) static_cast<float *>(p.out)[at + i * p.ldo] = glu_value(vs[i], us[i], p.form);
          else if (EPI == EPI_BF16) static_cast<bf16 *>(p.out)[at + i * p.ldo] = __float2bfloat16_rn(vs[i]);
          else static_cast<float *>(p.out)[at + i * p.ldo] = EPI == EPI_F32 ? vs[i] : olds[i] + vs[i];
        }
      }
    }
  }
}

template <int NX, bool LANES_A, int EPI, bool GROUPED, bool FUSED>
static cudaError_t allow() {
  return cudaFuncSetAttribute(gemm_fp8_few_kernel<NX, LANES_A, EPI, GROUPED, FUSED>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<NX, LANES_A, FUSED, GROUPED>::SMEM);
}

// How many CTAs in clusters of `split` the device holds at once.  The runtime counts one CTA a multiprocessor for a kernel that allocates tensor memory; there are
// PER_SM, two or, of experts' rows in sixteens, three (two: 148 tiles 4.6 us, 296 5.8, 444 9.6).
template <int NX, bool LANES_A, bool FUSED, bool GROUPED>
static int resident(int split) {
  static G2bPerDevice kept[MOST_SPLIT + 1];
  const int dev = g2b_current_device();
  if (dev >= 0 && kept[split].value[dev] > 0) return kept[split].value[dev];
  int clusters = 0, each = 0;
  if (allow<NX, LANES_A, EPI_F32, GROUPED, FUSED>() == cudaSuccess) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split), cfg.blockDim = dim3(Shape<NX, LANES_A, FUSED, GROUPED>::THREADS), cfg.dynamicSmemBytes = Shape<NX, LANES_A, FUSED, GROUPED>::SMEM;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = split, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr, cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&clusters, gemm_fp8_few_kernel<NX, LANES_A, EPI_F32, GROUPED, FUSED>, &cfg) != cudaSuccess) clusters = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, gemm_fp8_few_kernel<NX, LANES_A, EPI_F32, GROUPED, FUSED>, Shape<NX, LANES_A, FUSED, GROUPED>::THREADS,
                                                      Shape<NX, LANES_A, FUSED, GROUPED>::SMEM) != cudaSuccess)
      each = 0;
    if (each == 1) clusters *= Shape<NX, LANES_A, FUSED, GROUPED>::PER_SM;
  }
  const int n = clusters > 0 ? clusters * split : 1;
  if (dev >= 0) kept[split].value[dev] = n;
  return n;
}

template <int NX, bool LANES_A, int EPI, bool GROUPED, bool FUSED>
static int launch(const CUtensorMap &map_a, const CUtensorMap &map_w, Few p, cudaStream_t stream) {
  static G2bPerDevice configured;
  const int dev = g2b_current_device();
  if (dev < 0 || !configured.value[dev]) {
    const cudaError_t e = allow<NX, LANES_A, EPI, GROUPED, FUSED>();
    if (e != cudaSuccess) G2B_REFUSE("gemm_fp8_few: %d bytes of shared memory: %s", Shape<NX, LANES_A, FUSED, GROUPED>::SMEM, cudaGetErrorString(e));
    if (dev >= 0) configured.value[dev] = 1;
  }
  long long tiles_m = ((long long)p.M + Shape<NX, LANES_A, FUSED, GROUPED>::ROWS_A - 1) / Shape<NX, LANES_A, FUSED, GROUPED>::ROWS_A;
  if (GROUPED) tiles_m = tiles_m + p.n_experts < p.M ? tiles_m + p.n_experts : p.M;       // (a tile has a row at least)
  const long long tiles_n = (p.N + Shape<NX, LANES_A, FUSED, GROUPED>::ROWS_W - 1) / Shape<NX, LANES_A, FUSED, GROUPED>::ROWS_W;
  if ((!GROUPED && tiles_n > MOST_TILES_N) || tiles_m * p.split * (GROUPED ? tiles_n : 1) > INT32_MAX) G2B_REFUSE("gemm_fp8_few: %d x %d is too large for one launch", p.M, p.N);
  p.tiles_n = (int)tiles_n;
  const dim3 grid((unsigned)(tiles_m * p.split * (GROUPED ? tiles_n : 1)), GROUPED ? 1u : (unsigned)tiles_n);
  g2b_launch_cluster(gemm_fp8_few_kernel<NX, LANES_A, EPI, GROUPED, FUSED>, grid, dim3(Shape<NX, LANES_A, FUSED, GROUPED>::THREADS),
                     (size_t)Shape<NX, LANES_A, FUSED, GROUPED>::SMEM, stream, (unsigned)p.split, map_a, map_w, p);
  return g2b_check_launch("gemm_fp8_few");
}

template <int NX, bool LANES_A, bool FUSED>
static int pick(int epi, const CUtensorMap &map_a, const CUtensorMap &map_w, const Few &p, cudaStream_t stream) {
  if (p.n_experts) {
    switch (epi) {
      case EPI_F32: return launch<NX, LANES_A, EPI_F32, true, FUSED>(map_a, map_w, p, stream);
      case EPI_GATED_F32: return launch<NX, LANES_A, EPI_GATED_F32, true, FUSED>(map_a, map_w, p, stream);
    }
  } else {
    switch (epi) {
      case EPI_BF16: return launch<NX, LANES_A, EPI_BF16, false, FUSED>(map_a, map_w, p, stream);
      case EPI_F32: return launch<NX, LANES_A, EPI_F32, false, FUSED>(map_a, map_w, p, stream);
      case EPI_ADD_F32: return launch<NX, LANES_A, EPI_ADD_F32, false, FUSED>(map_a, map_w, p, stream);
      case EPI_GATED_F32: return launch<NX, LANES_A, EPI_GATED_F32, false, FUSED>(map_a, map_w, p, stream);
    }
  }
  G2B_REFUSE("gemm_fp8_few: no epilogue %d%s", epi, p.n_experts ? " for experts" : "");
}

// columns: 16, 32 or 64 rows of a side by side, or -64: 64 rows of w beside 128 of a; split: parts of K, at most 8.  With p.x (columns is 16 then): K a
// multiple of 8 and every row of x on 16 bytes.
static int run(const Product &given, int columns, int split, cudaStream_t stream) {
  if (given.x && (columns != 16 || given.K % 8 || given.x_stride % (given.x_f32 ? 4 : 8) || ((uintptr_t)given.x & 15) || given.top < 1))
    G2B_REFUSE("gemm_fp8_few: rows of %d values are not quantised on the way", given.K);
  if (given.idx && (!given.x || given.M > MOST_INLINE || given.n_experts < 1)) G2B_REFUSE("gemm_fp8_few: %d pairs are not sorted by the product", given.M);
  if (split < 1 || split > MOST_SPLIT) G2B_REFUSE("gemm_fp8_few: %d parts of K", split);
  CUtensorMap map_a, map_w;
  int rc = get_map(&map_w, given.w, given.w_rows(), given.blocks * BK, (int)given.ldw, columns < 0 ? 64 : LANES, 1);
  if (given.x) map_a = map_w;
  else if (!rc) rc = get_map(&map_a, given.a, given.M, given.blocks * BK, (int)given.lda, columns < 0 ? LANES : columns, 1);
  if (rc) G2B_REFUSE("gemm_fp8_few: cuTensorMapEncodeTiled failed (%d)", rc);
  Few p;
  static_cast<Product &>(p) = given;
  p.nb = given.scale_rows(), p.split = split;
  if (given.x) return pick<16, false, true>(given.epi, map_a, map_w, p, stream);
  switch (columns) {
    case 16: return pick<16, false, false>(given.epi, map_a, map_w, p, stream);
    case 32: return pick<32, false, false>(given.epi, map_a, map_w, p, stream);
    case 64: return pick<64, false, false>(given.epi, map_a, map_w, p, stream);
    case -64: return pick<64, true, false>(given.epi, map_a, map_w, p, stream);
  }
  G2B_REFUSE("gemm_fp8_few: no tiles of %d columns", columns);
}

}  // namespace few
