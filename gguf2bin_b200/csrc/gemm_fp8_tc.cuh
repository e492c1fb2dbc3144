// Products in 8-bit floating point (fp8.cuh) of many rows, on the 5th-generation tensor cores:
//   C[t, n] = sum_b s[b, t] S[n / 128, b] sum_{k in block b} q[t, k] Q[n, k].
//
// The scales change every 128 of K, so no accumulator can run over all of K: a block's sums are formed in tensor memory (four
// tcgen05.mma of kind::f8f6f4, M = N = 256, K = 32, a pair of CTAs) and added, times the two scales, to sums in registers.
// Roles by warp, a pair of CTAs a tile of 256 x 256 (each its own 128 rows), one pair after another of the persistent grid:
//   warp 8   copies: a block of K of the CTA's rows of A and of its half of W's 256 (128-byte swizzle), STAGES in flight
//   warp 9   products, in the pair's first CTA, into one of two accumulators of 256 columns
//   warps 0-7  add: warp w reads lanes 32 (w % 4) .. + 31 (a thread owns a row of A, so its scale is one number a block) and columns
//              128 (w / 4) .. + 127 (one block of W's rows: one number too) of a finished accumulator while the other one is filled;
//              behind the last block they write C, through shared memory, in rows
//
// `starts`: W is a stack of matrices and rows starts[e] .. starts[e + 1] of A meet the e-th.  Gated: rows of W alternate, eight gates and the eight
// ups of the same outputs, each with the scales of their own matrix; a tile is then 128 outputs wide, one block of the rows that the next product
// reads, so their scale is known where they are made.
//
// What bounds it: the sums' way out of tensor memory beside the products.  A block of K is 512 cycles of products and takes about 900 of the adders' round of
// waiting, loading and adding; the tensor pipe is busy 56 % of the time (8,192 rows by 4,096 x 12,288), DRAM 21 %, the issue slots 38 %.  Without the
// additions a block takes 640 to 690 cycles, and more of an accumulator on its way at once makes it longer (four pieces, or the next block's first ones
// behind this one's last: 3 to 8 % slower).  The walk over all of it then meets the power cap: 2,048 rows by 6,144 x 4,096 50 us cool and 55 hot (2,060 and
// 1,870 TFLOP/s), 8,192 by 4,096 x 12,288 added to a stream 382 and 441, gate and up of 17,408 x 5,120 at 2,048 rows 316 and 370 (2,310 and 1,970).
//
// Every wait on a barrier gives up after a bounded number of polls and leaves a code in `*status`, as in gemm_tc.cu; the allocation of tensor memory waits for
// CTAs that end whatever this one does (see tmem_alloc).
#pragma once
#include "product_fp8.cuh"

namespace many {

enum { ST_PRODUCER_TIMEOUT = 31, ST_MMA_TIMEOUT = 32, ST_ADDER_TIMEOUT = 33 };

constexpr int BM = 128, BN = 256, BK = F8_BLOCK;        // BM: rows of a CTA
constexpr int PART_BYTES = BM * BK, STAGE_BYTES = 2 * PART_BYTES;
constexpr int STAGES = 5;
constexpr int ADDERS = 8, THREADS = (ADDERS + 4) * 32;   // the last two warps only complete a group of four
// Registers: 384 threads start with 168 each (64,512); the adders hold 128 sums and two pieces of an accumulator and take 232, the others
// keep 40: 256 * 232 + 128 * 40 = 64,512.
constexpr int ADDER_REGS = 232, OTHER_REGS = 40;
constexpr int COLS = BN / 2, PIECE = 16;
constexpr int RING_BYTES = STAGES * STAGE_BYTES;
constexpr int BOX_BYTES = 32 * 128;                      // an adder's outputs on their way to C: 32 rows of 128 bytes, swizzled as the ring is
constexpr int BAR_BYTES = 256, TILE_BYTES = ADDERS * 16, LIST_BYTES = (2 * MOST_EXPERTS + 4) * 4;
// Boxes of an adder: two where there is room, so that one is filled while the other is written out.
template <bool GROUPED> constexpr int BOXES = GROUPED ? 1 : 2;
template <bool GROUPED>
constexpr int SMEM = RING_BYTES + ADDERS * BOXES<GROUPED> * BOX_BYTES + BAR_BYTES + TILE_BYTES + (GROUPED ? LIST_BYTES : 0) + 1024;      // + the swizzle's alignment
static_assert(SMEM<false> <= 227 * 1024 && SMEM<true> <= 227 * 1024, "one CTA a multiprocessor");
constexpr int BAND = 8;                                  // tiles along M that are walked side by side

struct Tc : Product {
  int nb, boxes, silu;                                   // nb: blocks of W's rows that have a scale; boxes: map_out may be used; silu: form is the plain one
};

template <bool ACC>
__device__ __forceinline__ void umma_f8_pair(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  constexpr uint32_t HIGH = (1024 >> 4) | (1u << 14) | (2u << 29);
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %4};\n\t"
      "mov.b64 db, {%2, %4};\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %3, p;\n\t}\n"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(HIGH), "n"(ACC ? 1 : 0)
      : "memory");
}
// Waits for this thread's loads of tensor memory; the registers pass through, so that nothing that reads them moves in front.
__device__ __forceinline__ void loaded32(uint32_t (&a)[16], uint32_t (&b)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" : F8_RW8(a, 0), F8_RW8(a, 8), F8_RW8(b, 0), F8_RW8(b, 8) : : "memory");
}
// One arrival on a barrier of the pair: this warp's reads of tensor memory are done (they are waited for); it hands over no data.
__device__ __forceinline__ void arrive_read(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_bar) : "memory");
}
// accumulator float, both operands e4m3 and K-major
constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(2 * BM >> 4) << 24);

struct Tile { int e, m0, end, n0; };

// Tile t of the walk.  `list` (in shared memory): with experts, list[e] = tiles of the experts up to e along M, and behind them p.starts.
template <bool GROUPED>
__device__ __forceinline__ Tile find_tile(const Tc &p, const int *list, int t, int tiles_n) {
  Tile r;
  if (GROUPED) {
    int lo = 0, hi = p.n_experts - 1;                    // the first expert with list[e] * tiles_n > t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (list[mid] * tiles_n > t) hi = mid;
      else lo = mid + 1;
    }
    const int before = lo ? list[lo - 1] : 0, high = list[lo] - before, at = t - before * tiles_n;
    r.e = lo, r.n0 = at / high * BN, r.m0 = list[MOST_EXPERTS + lo] + at % high * 2 * BM, r.end = list[MOST_EXPERTS + lo + 1];
  } else {
    const int tiles_m = (p.M + 2 * BM - 1) / (2 * BM), band = t / (BAND * tiles_n), high = min(BAND, tiles_m - band * BAND), at = t - band * BAND * tiles_n;
    r.e = 0, r.n0 = at / high * BN, r.m0 = (band * BAND + at % high) * 2 * BM, r.end = p.M;
  }
  return r;
}

template <int EPI, bool GROUPED>
__global__ void __launch_bounds__(THREADS, 1)
gemm_fp8_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out,
                   const __grid_constant__ Tc p) {
  constexpr bool GATED = EPI == EPI_GATED_F32 || EPI == EPI_GATED_ROWS;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  constexpr int OUT_BYTES = ADDERS * BOXES<GROUPED> * BOX_BYTES;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + RING_BYTES + OUT_BYTES);
  // a stage's `done` says both that its operands are free and that its sums are there (so there are at least as many stages as accumulators: an
  // adder has seen it before the stage's next products are issued).  A commit costs the tensor cores about 200 cycles: one a block, not two.
  const uint32_t full0 = smem_addr(bars), done0 = full0 + 8 * STAGES, sum_empty0 = done0 + 8 * STAGES;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 2);
  int4 *tiles = reinterpret_cast<int4 *>(smem + RING_BYTES + OUT_BYTES + BAR_BYTES);      // an adding warp's tile: its first row, end, first column
  int *list = reinterpret_cast<int *>(tiles + ADDERS);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t half = cluster_ctarank();               // the pair's first CTA issues its products
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);                       // in the first CTA, with both CTAs' bytes
      mbar_init(done0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) mbar_init(sum_empty0 + 8 * b, 2 * ADDERS);      // in the first CTA: both CTAs' adders
    mbar_init_fence();
  }
  if (warp == ADDERS + 1) {
    tmem_alloc_pair(smem_addr(tmem_slot), 2 * BN);
    pdl_launch();                                        // only now: see tmem_alloc
  }
  pdl_wait();
  const int tiles_n = (p.N + BN - 1) / BN;
  int n_tiles;
  if (GROUPED) {
    if (warp == 0) {                                     // tiles of the experts, summed up 32 at a time
      int sum = 0;
      for (int e0 = 0; e0 < p.n_experts; e0 += 32) {
        const int e = e0 + lane, first = p.starts[min(e, p.n_experts)], behind = p.starts[min(e + 1, p.n_experts)];
        int v = (behind - first + 2 * BM - 1) / (2 * BM);
        if (e <= p.n_experts) list[MOST_EXPERTS + e] = first;
        if (e + 1 == p.n_experts) list[MOST_EXPERTS + e + 1] = behind;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        if (e < p.n_experts) list[e] = sum + v;
        sum += __shfl_sync(0xffffffffu, v, 31);
      }
    }
  }
  tc_fence_before();
  cluster_sync_all();                                    // both CTAs' barriers, tensor memory and lists exist
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (GROUPED) n_tiles = list[p.n_experts - 1] * tiles_n;
  else n_tiles = (p.M + 2 * BM - 1) / (2 * BM) * tiles_n;
  const int pairs = gridDim.x / 2, pair = blockIdx.x / 2;

  if (warp >= ADDERS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(OTHER_REGS));
    // Both loops are walked by their whole warps, with one lane elected around what is issued: see elect_one.
    if (warp == ADDERS && PRODUCER_RUNS) {
      const uint32_t first_full0 = map_to_cta(full0, 0);
      bool ok = true;
      int it = 0;
      for (int t = pair; t < n_tiles && ok; t += pairs) {
        const Tile tile = find_tile<GROUPED>(p, list, t, tiles_n);
        const int row_a = tile.m0 + (int)half * BM, row_w = tile.e * p.N + tile.n0 + (int)half * BM;
        for (int b = 0; b < p.blocks; ++b, ++it) {
          const int s = it % STAGES;
          if (it >= STAGES) ok = __all_sync(0xffffffffu, mbar_wait(done0 + 8 * s, (it / STAGES - 1) & 1));
          if (!ok) {
            if (lane == 0) atomicExch(p.status, ST_PRODUCER_TIMEOUT);
            break;
          }
          const uint32_t to = smem_addr(smem + s * STAGE_BYTES);
          if (elect_one()) {
            if (half == 0) mbar_expect_tx(full0 + 8 * s, 2 * STAGE_BYTES);
            tma_load_2d_pair(to, &map_a, b * BK, row_a, first_full0 + 8 * s);
            tma_load_2d_pair(to + PART_BYTES, &map_w, b * BK, row_w, first_full0 + 8 * s);
          }
          __syncwarp();
        }
      }
    }
    if (warp == ADDERS + 1 && half == 0) {
      bool ok = true;
      int it = 0;
      for (int t = pair; t < n_tiles && ok; t += pairs)
        for (int b = 0; b < p.blocks; ++b, ++it) {
          const int s = it % STAGES, h = it & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, (it / STAGES) & 1) && (it < 2 || mbar_wait(sum_empty0 + 8 * h, (it / 2 - 1) & 1)));
          if (!ok) {
            if (lane == 0) atomicExch(p.status, ST_MMA_TIMEOUT);
            break;
          }
          tc_fence_after();
          const uint32_t lo = ((smem_addr(smem + s * STAGE_BYTES) & 0x3FFFF) >> 4) | 1u << 16;
          const uint32_t to = tmem + h * BN;
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (k == 0) umma_f8_pair<false>(to, lo, lo + PART_BYTES / 16, IDESC);
              else umma_f8_pair<true>(to, lo + 2 * k, lo + PART_BYTES / 16 + 2 * k, IDESC);
            }
            umma_commit_pair(done0 + 8 * s, 3);
          }
          __syncwarp();
        }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(ADDER_REGS));
    const int row0 = 32 * (warp % 4), col0 = COLS * (warp / 4);
    const uint32_t first_empty0 = map_to_cta(sum_empty0, 0);
    const uint32_t from0 = tmem + ((uint32_t)row0 << 16) + col0;
    unsigned char *const boxes = smem + RING_BYTES + warp * BOXES<GROUPED> * BOX_BYTES;
    int box = 0;
    bool ok = true;                                      // once a wait gave up nothing is waited for any more, and (but with EPI_GATED_ROWS, whose warps
    int it = 0;                                          // meet in pairs at every tile) nothing is written
    // Inside the loop over K the sums and the pieces of an accumulator take 160 of the 232 registers and addresses most of the rest: the tile waits in
    // shared memory, and the scales' places are 32-bit offsets.  A tile's first scales are asked for in front of the last one's outputs.
    int at_a = 0, at_w = 0;
    float next_a = 0.f, next_w = 0.f, next_up = 0.f;
    auto begin = [&](int t) {
      const Tile tile = find_tile<GROUPED>(p, list, t, tiles_n);
      const int m0 = tile.m0 + (int)half * BM + row0;
      at_a = min(m0 + lane, p.M - 1);
      // the thread's columns are one block of W's rows; gated, one of the gate's and one of the up's
      const int n_block = GATED ? tile.n0 / 2 / F8_BLOCK : min((tile.n0 + col0) / F8_BLOCK, p.nb - 1);
      at_w = (tile.e * (GATED ? 2 : 1) * p.nb + n_block) * p.blocks;
      next_a = p.sa[at_a], next_w = p.sw[at_w], next_up = GATED ? p.sw[at_w + p.nb * p.blocks] : 0.f;
      __syncwarp();
      if (lane == 0) tiles[warp] = make_int4(m0, tile.end, tile.n0, 0);
      __syncwarp();
    };
    if (pair < n_tiles) begin(pair);
    for (int t = pair; t < n_tiles; t += pairs) {
      float sum[COLS];
#pragma unroll
      for (int j = 0; j < COLS; ++j) sum[j] = 0.f;
      for (int b = 0; b < p.blocks; ++b, ++it) {
        const int h = it & 1;
        const float f = next_a * next_w, f_up = next_a * next_up;
        if (b + 1 < p.blocks) {
          at_a += (int)p.lds, ++at_w;
          next_a = p.sa[at_a];
          next_w = p.sw[at_w];
          if (GATED) next_up = p.sw[at_w + p.nb * p.blocks];
        }
        if (!ok) continue;
        ok = __all_sync(0xffffffffu, mbar_wait(done0 + 8 * (it % STAGES), (it / STAGES) & 1));      // the warp's lanes agree: its loads are all lanes'
        if (!ok) {
          if (lane == 0) atomicExch(p.status, ST_ADDER_TIMEOUT);
          continue;
        }
        tc_fence_after();
        // Two pieces of 16 columns are on their way while two are added.  (Of 32 columns the loop kept sums in memory: 380 -> 560 us.)
        uint32_t x[2][PIECE];
        auto add = [&](int c, const uint32_t (&v)[PIECE]) {
#pragma unroll
          for (int j = 0; j < PIECE; j += 2) {
            const float fj = GATED && (j & 8) ? f_up : f;
            const float2 s = fma2(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), make_float2(fj, fj), make_float2(sum[c + j], sum[c + j + 1]));
            sum[c + j] = s.x, sum[c + j + 1] = s.y;
          }
        };
        const uint32_t from = from0 + h * BN;
        tmem_ld16(from, x[0]);
        tmem_ld16(from + 16, x[1]);
#pragma unroll
        for (int c = 0; c < COLS; c += 32) {
          loaded32(x[0], x[1]);
          if (c + 32 == COLS) {                          // the accumulator is read: its next products need not wait for these sums
            tc_fence_before();
            __syncwarp();
            if (lane == 0) arrive_read(first_empty0 + 8 * h);
          }
          add(c, x[0]);
          if (c + 32 < COLS) tmem_ld16(from + c + 32, x[0]);
          add(c + 16, x[1]);
          if (c + 32 < COLS) tmem_ld16(from + c + 48, x[1]);
        }
      }
      if (!ok && EPI != EPI_GATED_ROWS) break;
      const int4 tile = tiles[warp];
      const int m0 = tile.x, n0 = tile.z;
      if (t + pairs < n_tiles) begin(t + pairs);
      const int rows = min(32, tile.y - m0);           // of this warp's that exist (may be none)
      if (GATED) {
        const int n_out = p.N / 2, out0 = (n0 + col0) / 2;                        // 64 outputs a thread
        [[maybe_unused]] float most = 0.f;
        // (what is left in float has 32 bits' precision; the fast forms, within 2^-20 or so, where four bits of it are kept)
        constexpr bool FAST = EPI == EPI_GATED_ROWS;
        if (p.silu) {
#pragma unroll
          for (int j = 0; j < COLS / 2; ++j) {
            const float g = sum[(j >> 3) * 16 + (j & 7)], u = sum[(j >> 3) * 16 + (j & 7) + 8];
            sum[j] = FAST ? silu_value_fast(g, u) : silu_value(g, u);
          }
        } else {
#pragma unroll
          for (int j = 0; j < COLS / 2; ++j) {
            const float g = sum[(j >> 3) * 16 + (j & 7)], u = sum[(j >> 3) * 16 + (j & 7) + 8];
            sum[j] = FAST ? glu_value_fast(g, u, p.form) : glu_value(g, u, p.form);
          }
        }
        if (out0 + COLS / 2 > n_out)                     // the last outputs' tile: zeros behind them
#pragma unroll
          for (int j = 0; j < COLS / 2; ++j)
            if (out0 + j >= n_out) sum[j] = 0.f;
        if (EPI == EPI_GATED_ROWS) {
          float *const given = reinterpret_cast<float *>(boxes + BOX_BYTES / 2);       // the largest of a row: of the two warps that share it
#pragma unroll
          for (int j = 0; j < COLS / 2; ++j) most = max_nan(most, fabsf(sum[j]));
          given[lane] = most;
          asm volatile("bar.sync %0, 64;\n" ::"r"(1 + warp % 4) : "memory");
          most = max_nan(most, (given + (warp < 4 ? 4 : -4) * BOXES<GROUPED> * BOX_BYTES / 4)[lane]);
          const BlockScale s = block_scale(most);
          if (lane < rows && warp < 4) p.out_scale[n0 / 2 / F8_BLOCK * p.ldos + m0 + lane] = s.scale;
          // 64 bytes a row, in rows through a box (the copy unit does not know an expert's last row, so there lanes write their own)
          const bool copied = p.boxes && (!GROUPED || rows == 32);
          if (copied && lane == 0) bulk_wait_read<0>();
          __syncwarp();
          uint8_t *const to = static_cast<uint8_t *>(p.out) + (long long)(m0 + lane) * p.ldo + out0;
#pragma unroll
          for (int j = 0; j < COLS / 2; j += 16) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = pack_e4m3(sum[j + 4 * i] * s.inverse, sum[j + 4 * i + 1] * s.inverse, sum[j + 4 * i + 2] * s.inverse, sum[j + 4 * i + 3] * s.inverse);
            if (copied) *reinterpret_cast<uint4 *>(boxes + lane * 64 + ((j / 16 ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            else if (lane < rows) *reinterpret_cast<uint4 *>(to + j) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (copied) {
            fence_async_shared();
            __syncwarp();
            if (lane == 0 && rows > 0) {
              tma_store_2d(&map_out, smem_addr(boxes), out0, m0);
              bulk_commit();
            }
          }
          asm volatile("bar.sync %0, 64;\n" ::"r"(1 + warp % 4) : "memory");     // the next tile's largest go where this one's were
          continue;
        }
      }
      if (rows <= 0) continue;
      // 32 rows of 128 bytes at a time through a box: written out (or added to what is there: every output gets one addition) by the copy unit,
      // or, where C's rows do not start on 16 bytes or some of the rows are another expert's, read back by the warp.
      constexpr int OUTS = GATED ? COLS / 2 : COLS, WIDE = EPI == EPI_BF16 ? 64 : 32;
      const int n_out = GATED ? p.N / 2 : p.N, first = GATED ? (n0 + col0) / 2 : n0 + col0;
      // (the copy unit cuts a row off at 16 bytes only: what lies behind C's last column may be another's)
      const bool cut = n_out % (EPI == EPI_BF16 ? 8 : 4) != 0;
#pragma unroll
      for (int q = 0; q < OUTS / WIDE; ++q) {
        const int n1 = first + WIDE * q;
        if (n1 >= n_out) break;
        const bool copied = p.boxes && (!GROUPED || rows == 32) && !(cut && n1 + WIDE > n_out);
        int l = lane;
        asm volatile("" : "+r"(l));                      // or the boxes' addresses are kept over the loop above
        unsigned char *const at = boxes + box * BOX_BYTES;
        box = (box + 1) % BOXES<GROUPED>;
        if (lane == 0) bulk_wait_read<BOXES<GROUPED> - 1>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int c = WIDE * q + WIDE / 8 * j;
          uint4 w;
          if (EPI == EPI_BF16) {
            uint32_t u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const __nv_bfloat162 pair2 = __floats2bfloat162_rn(sum[c + 2 * i], sum[c + 2 * i + 1]);
              u[i] = *reinterpret_cast<const uint32_t *>(&pair2);
            }
            w = make_uint4(u[0], u[1], u[2], u[3]);
          } else {
            w = make_uint4(__float_as_uint(sum[c]), __float_as_uint(sum[c + 1]), __float_as_uint(sum[c + 2]), __float_as_uint(sum[c + 3]));
          }
          *reinterpret_cast<uint4 *>(at + l * 128 + ((j ^ (l & 7)) << 4)) = w;
        }
        if (copied) {
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            if (EPI == EPI_ADD_F32) tma_reduce_add_2d(&map_out, smem_addr(at), n1, m0);
            else tma_store_2d(&map_out, smem_addr(at), n1, m0);
            bulk_commit();
          }
        } else if (p.boxes && n1 + WIDE <= n_out) {      // (of an expert's last rows; nothing is added to there)
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + lane / 8, j = lane % 8;
            if (r >= rows) break;
            *reinterpret_cast<uint4 *>(static_cast<unsigned char *>(p.out) + ((long long)(m0 + r) * p.ldo + n1 + WIDE / 8 * j) * (EPI == EPI_BF16 ? 2 : 4)) =
                *reinterpret_cast<const uint4 *>(at + r * 128 + ((j ^ (r & 7)) << 4));
          }
          __syncwarp();
        } else {
          // rows that start anywhere: neighbouring lanes neighbouring outputs of a row (2,115 rows by 7,079 x 4,046 into a stream
          // 140 us, eight rows at a time 152, four neighbours a lane 218; by 7,080 89)
          if (lane == 0) bulk_commit();                  // (nothing: boxes are counted by their groups)
          __syncwarp();
          constexpr int SIZE = EPI == EPI_BF16 ? 2 : 4, EACH = 16 / SIZE, ROWS = 16;
#pragma unroll
          for (int c = lane; c < WIDE; c += 32) {
            if (n1 + c >= n_out) break;
            unsigned char *to = static_cast<unsigned char *>(p.out) + ((long long)m0 * p.ldo + n1 + c) * SIZE;
            for (int r0 = 0; r0 < rows; r0 += ROWS) {
              float old[ROWS];
#pragma unroll
              for (int i = 0; i < ROWS; ++i) old[i] = EPI == EPI_ADD_F32 && r0 + i < rows ? *reinterpret_cast<const float *>(to + (r0 + i) * p.ldo * SIZE) : 0.f;
#pragma unroll
              for (int i = 0; i < ROWS; ++i) {
                const int r = r0 + i;
                if (r >= rows) break;
                const unsigned char *v = at + r * 128 + ((c / EACH ^ (r & 7)) << 4) + c % EACH * SIZE;
                if (EPI == EPI_BF16) *reinterpret_cast<uint16_t *>(to + r * p.ldo * SIZE) = *reinterpret_cast<const uint16_t *>(v);
                else if (EPI == EPI_ADD_F32) *reinterpret_cast<float *>(to + r * p.ldo * SIZE) = old[i] + *reinterpret_cast<const float *>(v);
                else *reinterpret_cast<float *>(to + r * p.ldo * SIZE) = *reinterpret_cast<const float *>(v);
              }
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait<0>();                       // what the copy unit still reads and writes
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();                                    // neither CTA's products, copies and arrivals meet a peer that is gone
  if (warp == ADDERS + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 2 * BN);
  }
}

// How many pairs the device holds at once.
template <int EPI, bool GROUPED>
static int most_pairs() {
  static G2bPerDevice kept;
  const int dev = g2b_current_device();
  if (dev >= 0 && kept.value[dev] > 0) return kept.value[dev];
  const int smem = SMEM<GROUPED>;
  if (cudaFuncSetAttribute(gemm_fp8_tc_kernel<EPI, GROUPED>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2), cfg.blockDim = dim3(THREADS), cfg.dynamicSmemBytes = (size_t)smem;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, gemm_fp8_tc_kernel<EPI, GROUPED>, &cfg) != cudaSuccess) n = 0;
  if (dev >= 0) kept.value[dev] = n;
  return n;
}

template <int EPI, bool GROUPED>
static int launch(const CUtensorMap &map_a, const CUtensorMap &map_w, Tc p, cudaStream_t stream) {
  const int most = most_pairs<EPI, GROUPED>();
  if (most < 1) G2B_REFUSE("gemm_fp8_tc: the device holds no pair with %d bytes of shared memory", SMEM<GROUPED>);
  const long long tiles_n = (p.N + BN - 1) / BN;
  const long long tiles = GROUPED ? most : ((long long)p.M + 2 * BM - 1) / (2 * BM) * tiles_n;
  if (((long long)p.M / (2 * BM) + 1 + (GROUPED ? p.n_experts : 0)) * tiles_n > INT32_MAX) G2B_REFUSE("gemm_fp8_tc: %d x %d is too large for one launch", p.M, p.N);
  const int pairs = (int)(tiles < most ? tiles : most);
  CUtensorMap map_out = map_a;
  constexpr bool ROWS = EPI == EPI_GATED_ROWS;
  constexpr int SIZE = ROWS ? 1 : EPI == EPI_BF16 ? 2 : 4;
  p.boxes = p.ldo * SIZE % 16 == 0 && ((uintptr_t)p.out & 15) == 0 && p.ldo <= INT32_MAX;
  p.silu = p.form.limit == INFINITY && p.form.offset == 0.f && p.form.c1 == 1.f && p.form.c3 == 0.f;
  if (p.boxes) {                                         // (quantised rows go to their blocks' ends, zeros included)
    const int columns = ROWS ? (p.N / 2 + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK : EPI == EPI_GATED_F32 ? p.N / 2 : p.N;
    const int rc = get_map(&map_out, p.out, p.M, columns, (int)p.ldo, 32, SIZE, ROWS ? 64 : 128);
    if (rc) G2B_REFUSE("gemm_fp8_tc: cuTensorMapEncodeTiled failed (%d)", rc);
  }
  g2b_launch_cluster(gemm_fp8_tc_kernel<EPI, GROUPED>, dim3(2 * pairs), dim3(THREADS), (size_t)SMEM<GROUPED>, stream, 2u, map_a, map_w, map_out, p);
  return g2b_check_launch("gemm_fp8_tc");
}

static int resident() { return most_pairs<EPI_F32, false>() > 0 ? most_pairs<EPI_F32, false>() : 1; }

static int run(const Product &given, cudaStream_t stream) {
  const long long w_rows = given.w_rows();
  if ((w_rows / F8_BLOCK + 2ll * given.n_experts + 2) * given.blocks > INT32_MAX || given.lds * given.blocks > INT32_MAX)
    G2B_REFUSE("gemm_fp8_tc: %d rows of A and %lld of W with %d blocks are too many for one launch", given.M, w_rows, given.blocks);
  CUtensorMap map_a, map_w;
  int rc = get_map(&map_a, given.a, given.M, given.blocks * BK, (int)given.lda, BM, 1);
  if (!rc) rc = get_map(&map_w, given.w, w_rows, given.blocks * BK, (int)given.ldw, BM, 1);
  if (rc) G2B_REFUSE("gemm_fp8_tc: cuTensorMapEncodeTiled failed (%d)", rc);
  Tc p;
  static_cast<Product &>(p) = given;
  p.nb = given.scale_rows();
  if (given.n_experts) {
    switch (given.epi) {
      case EPI_F32: return launch<EPI_F32, true>(map_a, map_w, p, stream);
      case EPI_GATED_ROWS: return launch<EPI_GATED_ROWS, true>(map_a, map_w, p, stream);
    }
  } else {
    switch (given.epi) {
      case EPI_BF16: return launch<EPI_BF16, false>(map_a, map_w, p, stream);
      case EPI_F32: return launch<EPI_F32, false>(map_a, map_w, p, stream);
      case EPI_ADD_F32: return launch<EPI_ADD_F32, false>(map_a, map_w, p, stream);
      case EPI_GATED_F32: return launch<EPI_GATED_F32, false>(map_a, map_w, p, stream);
      case EPI_GATED_ROWS: return launch<EPI_GATED_ROWS, false>(map_a, map_w, p, stream);
    }
  }
  G2B_REFUSE("gemm_fp8_tc: no epilogue %d%s", given.epi, given.n_experts ? " for experts" : "");
}

}  // namespace many
