// What stands around the products in 8-bit floating point (fp8.cuh):
//
//   quantize_rows    rows of activations: a scale for every row and 128 columns.  q [T, blocks * 128] (zeros behind K), scale [blocks, T], rows
//                    innermost, because a product's thread owns a row and the lanes of a warp own neighbours.  With `pair_row` a row goes to the
//                    places of its `top` choices instead (see moe_sort): read and quantised once, written `top` times.
//   quantize_matrix  a matrix, or a stack of them: a scale for every 128 x 128.
//   moe_sort         the (token, choice) pairs in the order of their experts, stable: pairs of one expert keep their order, so a row's place depends on
//                    the choices alone.  starts[e] .. starts[e + 1]: the rows of expert e.  Pairs of experts from `n_real` on get no row (-1).
//   moe_back         y_t = sum_j weight_tj (row of pair (t, j), or the token's own input where the pair has none), in the order of j.
//
// (moe.cu has both for experts of other types: moe_plan lists tiles for its products and gives places as its atomics fall, where here rows are quantised and
// compared by place; moe_combine reads and stores float of any width, moe_back either type four values at a time.)
//
// All are bound by their bytes, or by their launch: 8,192 x 4,096 bfloat16 in 20.6 us (4.9 TB/s read and written), float 28 (6.0), 8,192 x 12,288 bfloat16 59;
// 16,384 pairs sorted in 10.5 us, 4,096 rows of 2,048 to four places each 9.7, and back with weights 24.5 (5.6 TB/s).
#pragma once
#include "fp8.cuh"

// ---- four values ---------------------------------------------------------------------------------------
__device__ __forceinline__ float4 load4(const float *p) { return *reinterpret_cast<const float4 *>(p); }
__device__ __forceinline__ float4 load4(const bf16 *p) {
  const uint2 w = *reinterpret_cast<const uint2 *>(p);
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
}

// ---- rows -------------------------------------------------------------------------------------------------
// Eight values of a row from column k on; zeros behind K.  VEC = 8: every row on 16 bytes and K a multiple of 8; 4: the same of fours (bfloat16: on 8
// bytes); 1: anything.
template <typename T, int VEC>
__device__ __forceinline__ void load8(const T *x, int k, int K, float (&v)[8]) {
  if (VEC == 8 && sizeof(T) == 2) {
    const uint4 a = k < K ? *reinterpret_cast<const uint4 *>(x + k) : make_uint4(0, 0, 0, 0);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  } else if (VEC >= 4) {
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
      const float4 a = k + h < K ? load4(x + k + h) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[h] = a.x, v[h + 1] = a.y, v[h + 2] = a.z, v[h + 3] = a.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? to_f32(x[k + i]) : 0.f;
  }
}

constexpr int ROWS_AT_ONCE = 16, BLOCKS_AT_ONCE = 4;

// Sixteen lanes a row, eight values each; a block of threads takes 16 rows x 4 blocks of 128.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T *__restrict__ x, long long x_stride, int tokens, int K, int blocks, uint8_t *__restrict__ q, long long q_stride,
                     float *__restrict__ scale, long long scale_stride, const int *__restrict__ pair_row, int top, int n_rows) {
  pdl_launch();
  const int lane = threadIdx.x & 15;
  const long long t = (long long)blockIdx.x * ROWS_AT_ONCE + (threadIdx.x >> 4);
  const int b0 = blockIdx.y * BLOCKS_AT_ONCE;
  pdl_wait();
  if (t >= tokens) return;                       // (sixteen lanes of a warp may leave: the shuffles below stay among sixteen)
  const uint32_t among = 0xffffu << (threadIdx.x & 16);
  float v[BLOCKS_AT_ONCE][8];
#pragma unroll
  for (int u = 0; u < BLOCKS_AT_ONCE; ++u) load8<T, VEC>(x + t * x_stride, (b0 + u) * F8_BLOCK + 8 * lane, K, v[u]);
#pragma unroll
  for (int u = 0; u < BLOCKS_AT_ONCE; ++u) {
    if (b0 + u >= blocks) break;
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(v[u][i]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(among, m, o, 16));
    const BlockScale s = block_scale(m);
    const float f = s.inverse;
    const uint2 w = make_uint2(pack_e4m3(v[u][0] * f, v[u][1] * f, v[u][2] * f, v[u][3] * f), pack_e4m3(v[u][4] * f, v[u][5] * f, v[u][6] * f, v[u][7] * f));
    const int at = (b0 + u) * F8_BLOCK + 8 * lane;
    if (!pair_row) {
      *reinterpret_cast<uint2 *>(q + t * q_stride + at) = w;
      if (lane == 0) scale[(b0 + u) * scale_stride + t] = s.scale;
    } else {
      for (int j = 0; j < top; ++j) {
        const int r = pair_row[t * top + j];
        if (r < 0 || r >= n_rows) continue;
        *reinterpret_cast<uint2 *>(q + r * q_stride + at) = w;
        if (lane == 0) scale[(b0 + u) * scale_stride + r] = s.scale;
      }
    }
  }
}

template <typename T>
static void launch_rows(int vec, dim3 grid, cudaStream_t stream, const void *x, long long x_stride, int tokens, int K, int blocks, void *q,
                        long long q_stride, float *scale, long long scale_stride, const int *pair_row, int top, int n_rows) {
  g2b_launch(vec == 8 ? quantize_rows_kernel<T, 8> : vec == 4 ? quantize_rows_kernel<T, 4> : quantize_rows_kernel<T, 1>, grid, dim3(256), 0, stream, (const T *)x, x_stride, tokens, K,
             blocks, (uint8_t *)q, q_stride, scale, scale_stride, pair_row, top, n_rows);
}

// pair_row: int [tokens * top], or null (then every row of x has a row of q, and top is 1); places outside 0 .. n_rows - 1 are left out.  No choices
// (top 0, whose places have no address either): nothing is written.  q's rows on 16 bytes.
static int run_quantize_rows(const void *x, int dtype, long long x_stride, int tokens, int K, void *q, long long q_stride, float *scale,
                                 long long scale_stride, const int *pair_row, int top, int n_rows, cudaStream_t stream) {
  if (tokens <= 0 || K <= 0 || top <= 0) return 0;
  const int blocks = (K + F8_BLOCK - 1) / F8_BLOCK;
  if (q_stride % 16 || q_stride < (long long)blocks * F8_BLOCK || ((uintptr_t)q & 15))
    G2B_REFUSE("quantize_rows: rows of q start on 16 bytes and hold %d blocks of %d", blocks, F8_BLOCK);
  const int steps = (blocks + BLOCKS_AT_ONCE - 1) / BLOCKS_AT_ONCE;
  if (steps > 65535) G2B_REFUSE("quantize_rows: K=%d is too large", K);
  const dim3 grid((unsigned)((tokens + ROWS_AT_ONCE - 1) / ROWS_AT_ONCE), (unsigned)steps);
  const int whole = (K | (int)(x_stride & 7)) & 7, odd = (int)((uintptr_t)x & 15);
  const int vec = whole == 0 && odd == 0 ? 8 : whole % 4 == 0 && (dtype == G2B_F32 ? odd == 0 : odd % 8 == 0) ? 4 : 1;
  if (dtype == G2B_F32)
    launch_rows<float>(vec, grid, stream, x, x_stride, tokens, K, blocks, q, q_stride, scale, scale_stride, pair_row, top, n_rows);
  else if (dtype == G2B_BF16)
    launch_rows<bf16>(vec, grid, stream, x, x_stride, tokens, K, blocks, q, q_stride, scale, scale_stride, pair_row, top, n_rows);
  else
    G2B_REFUSE("quantize_rows: unknown dtype %d", dtype);
  return g2b_check_launch("quantize_rows");
}

// ---- matrices ---------------------------------------------------------------------------------------------
// A block of threads a block of 128 x 128 of one matrix of the stack; it is read twice (the second time from the L2).
template <typename T>
__global__ void __launch_bounds__(256)
quantize_matrix_kernel(const T *__restrict__ w, int N, int K, long long w_stride, uint8_t *__restrict__ q, long long q_stride, float *__restrict__ scale) {
  // (no early start for what follows: a product reads its matrix before it waits for the kernel in front of it)
  __shared__ float most[8];
  const int kb = blockIdx.x, nb = blockIdx.y;
  const long long e = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int k = kb * F8_BLOCK + 4 * lane, rows = min(F8_BLOCK, N - nb * F8_BLOCK);
  const T *from = w + (e * N + nb * F8_BLOCK) * w_stride;
  uint8_t *to = q + (e * N + nb * F8_BLOCK) * q_stride;
  pdl_wait();
  float m = 0.f;
  for (int r = warp; r < rows; r += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i < K) m = max_nan(m, fabsf(to_f32(from[r * w_stride + k + i])));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) most[warp] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max_nan(m, most[i]);
  const BlockScale s = block_scale(m);
  if (threadIdx.x == 0) scale[(e * gridDim.y + nb) * gridDim.x + kb] = s.scale;
  for (int r = warp; r < rows; r += 8) {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < K ? to_f32(from[r * w_stride + k + i]) * s.inverse : 0.f;
    *reinterpret_cast<uint32_t *>(to + r * q_stride + k) = pack_e4m3(v[0], v[1], v[2], v[3]);
  }
}

// `count` matrices [N, K] one behind the other (`w_stride`, `q_stride`: from row to row); scale [count, ceil(N / 128), ceil(K / 128)].
static int run_quantize_matrix(const void *w, int dtype, int count, int N, int K, long long w_stride, void *q, long long q_stride, float *scale,
                                   cudaStream_t stream) {
  if (count <= 0 || N <= 0 || K <= 0) return 0;
  const int kb = (K + F8_BLOCK - 1) / F8_BLOCK, nb = (N + F8_BLOCK - 1) / F8_BLOCK;
  if (q_stride % 16 || q_stride < (long long)kb * F8_BLOCK || ((uintptr_t)q & 15))
    G2B_REFUSE("quantize_matrix: rows of q start on 16 bytes and hold %d blocks of %d", kb, F8_BLOCK);
  if (nb > 65535 || count > 65535) G2B_REFUSE("quantize_matrix: %d matrices of %d rows are too many for one launch", count, N);
  const dim3 grid((unsigned)kb, (unsigned)nb, (unsigned)count);
  if (dtype == G2B_F32)
    g2b_launch(quantize_matrix_kernel<float>, grid, dim3(256), 0, stream, (const float *)w, N, K, w_stride, (uint8_t *)q, q_stride, scale);
  else if (dtype == G2B_BF16)
    g2b_launch(quantize_matrix_kernel<bf16>, grid, dim3(256), 0, stream, (const bf16 *)w, N, K, w_stride, (uint8_t *)q, q_stride, scale);
  else
    G2B_REFUSE("quantize_matrix: unknown dtype %d", dtype);
  return g2b_check_launch("quantize_matrix");
}

// ---- pairs by expert --------------------------------------------------------------------------------------
constexpr int SORT_WARPS = 32, SORT_AHEAD = 8;
static_assert(MOST_EXPERTS <= SORT_WARPS * 32, "an expert a thread");

// One block.  A warp takes a stretch of the pairs, 32 at a time: lanes with one expert find each other (a ballot a bit of its number: match.any
// takes 48 cycles of the multiprocessor: 27 us for 16,384 pairs, where this takes 12), the first of them counts for all.  No two warps share a counter, so
// nothing depends on who comes first.  A pair's place among its warp's waits in pair_row for the rows in front of it.
__global__ void __launch_bounds__(SORT_WARPS * 32)
moe_sort_kernel(const int *__restrict__ idx, int n_pairs, int n_real, int bits, int *__restrict__ starts, int *pair_row, int *__restrict__ row_pair) {
  extern __shared__ int at[];                    // [SORT_WARPS][n_real]: a warp's count of an expert, then the first row of its stretch
  __shared__ int warp_sum[SORT_WARPS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch();
  for (int i = threadIdx.x; i < SORT_WARPS * n_real; i += blockDim.x) at[i] = 0;
  const int per = (n_pairs + SORT_WARPS * 32 - 1) / (SORT_WARPS * 32) * 32;
  const int first = min(n_pairs, warp * per), last = min(n_pairs, first + per);
  pdl_wait();
  __syncthreads();
  int *own = at + warp * n_real;
  for (int p0 = first; p0 < last; p0 += 32 * SORT_AHEAD) {
    int e[SORT_AHEAD];
#pragma unroll
    for (int u = 0; u < SORT_AHEAD; ++u) e[u] = p0 + 32 * u + lane < last ? idx[p0 + 32 * u + lane] : -1;
#pragma unroll
    for (int u = 0; u < SORT_AHEAD; ++u) {
      const int p = p0 + 32 * u + lane;
      if (p0 + 32 * u >= last) break;
      const bool real = e[u] >= 0 && e[u] < n_real;
      uint32_t same = __ballot_sync(0xffffffffu, real);
      for (int b = 0; b < bits; ++b) {
        const uint32_t set = __ballot_sync(0xffffffffu, e[u] >> b & 1);
        same &= e[u] >> b & 1 ? set : ~set;
      }
      const uint32_t before = same & ((1u << lane) - 1);
      const int count = real ? own[e[u]] : 0;
      if (p < last) pair_row[p] = real ? count + __popc(before) : -1;
      __syncwarp();
      if (real && !before) own[e[u]] = count + __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  // rows of the experts before thread e's: a scan over the block, an expert a thread
  int total = 0;
  if (threadIdx.x < n_real)
    for (int w = 0; w < SORT_WARPS; ++w) total += at[w * n_real + threadIdx.x];
  int before = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) warp_sum[warp] = before;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sum[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    warp_sum[lane] = s;
  }
  __syncthreads();
  before += (warp ? warp_sum[warp - 1] : 0) - total;
  if (threadIdx.x < n_real) {
    starts[threadIdx.x] = before;
    if (threadIdx.x == n_real - 1) starts[n_real] = before + total;
    for (int w = 0; w < SORT_WARPS; ++w) {
      const int n = at[w * n_real + threadIdx.x];
      at[w * n_real + threadIdx.x] = before;
      before += n;
    }
  }
  __syncthreads();
#pragma unroll 4
  for (int p = first + lane; p < last; p += 32) {
    const int rank = pair_row[p];
    if (rank < 0) continue;
    const int row = own[idx[p]] + rank;
    pair_row[p] = row;
    if (row_pair) row_pair[row] = p;
  }
}

// starts: int [n_real + 1]; row_pair (the pair of every row in use) may be null
static int run_moe_sort(const int *idx, int n_pairs, int n_real, int *starts, int *pair_row, int *row_pair, cudaStream_t stream) {
  if (n_real < 1 || n_real > MOST_EXPERTS) G2B_REFUSE("moe_sort: %d experts outside 1..%d", n_real, MOST_EXPERTS);
  static G2bPerDevice configured;
  const int dev = g2b_current_device();
  if (dev < 0 || !configured.value[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(moe_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SORT_WARPS * MOST_EXPERTS * 4);
    if (e != cudaSuccess) G2B_REFUSE("moe_sort: %s", cudaGetErrorString(e));
    if (dev >= 0) configured.value[dev] = 1;
  }
  g2b_launch(moe_sort_kernel, dim3(1), dim3(SORT_WARPS * 32), (size_t)SORT_WARPS * n_real * 4, stream, idx, max(n_pairs, 0), n_real,
             n_real > 1 ? 32 - __builtin_clz(n_real - 1) : 0, starts, pair_row, row_pair);
  return g2b_check_launch("moe_sort");
}

// ---- back to the tokens -----------------------------------------------------------------------------------
// Four neighbours a thread; H a multiple of 4.
template <typename TSELF, typename TOUT, bool ACCUM>
__global__ void __launch_bounds__(256)
moe_back_kernel(const float *__restrict__ rows, const int *__restrict__ pair_row, const float *__restrict__ weight, const TSELF *__restrict__ x_self,
                long long self_stride, int n_rows, int top, int H, TOUT *__restrict__ out, long long out_stride) {
  pdl_launch();
  const long long t = blockIdx.x;
  const int c = 4 * (blockIdx.y * blockDim.x + threadIdx.x);
  pdl_wait();
  if (c >= H) return;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  constexpr int AHEAD = 4;
  for (int j0 = 0; j0 < top; j0 += AHEAD) {
    float4 v[AHEAD];
    float w[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (j0 + u >= top) break;
      const int r = pair_row[t * top + j0 + u];
      w[u] = weight[t * top + j0 + u];
      v[u] = r >= 0 && r < n_rows ? load4(rows + (long long)r * H + c) : load4(x_self + t * self_stride + c);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (j0 + u >= top) break;
      y.x = fmaf(w[u], v[u].x, y.x), y.y = fmaf(w[u], v[u].y, y.y), y.z = fmaf(w[u], v[u].z, y.z), y.w = fmaf(w[u], v[u].w, y.w);
    }
  }
  TOUT *to = out + t * out_stride + c;
  if constexpr (sizeof(TOUT) == 4) {
    if (ACCUM) {
      const float4 old = load4(to);
      y = make_float4(old.x + y.x, old.y + y.y, old.z + y.z, old.w + y.w);
    }
    *reinterpret_cast<float4 *>(to) = y;
  } else {
    const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
    *reinterpret_cast<uint2 *>(to) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
  }
}

template <typename TSELF, typename TOUT, bool ACCUM>
static void launch_back(int tokens, cudaStream_t stream, const float *rows, const int *pair_row, const float *weight, const void *x_self,
                        long long self_stride, int n_rows, int top, int H, void *out, long long out_stride) {
  const int threads = H >= 1024 ? 256 : 64;
  g2b_launch(moe_back_kernel<TSELF, TOUT, ACCUM>, dim3((unsigned)tokens, (unsigned)((H / 4 + threads - 1) / threads)), dim3(threads), 0, stream, rows,
             pair_row, weight, (const TSELF *)x_self, self_stride, n_rows, top, H, (TOUT *)out, out_stride);
}

// rows float [n_rows, H], x_self of `self_dtype`, out of `out_dtype`; everything on 16 bytes (bfloat16: 8), H and the strides multiples of 4.
static int run_moe_back(const float *rows, const int *pair_row, const float *weight, const void *x_self, int self_dtype, long long self_stride,
                            int n_rows, int tokens, int top, int H, void *out, int out_dtype, long long out_stride, int accumulate, cudaStream_t stream) {
  if (tokens <= 0 || H <= 0) return 0;
  if (H % 4 || self_stride % 4 || out_stride % 4 || ((uintptr_t)rows & 15) || ((uintptr_t)x_self & (self_dtype == G2B_F32 ? 15 : 7)) ||
      ((uintptr_t)out & (out_dtype == G2B_F32 ? 15 : 7)))
    G2B_REFUSE("moe_back: rows of %d values with strides (%lld, %lld) are not on 16 bytes", H, self_stride, out_stride);
  if (H / 4 > 65535 * 64) G2B_REFUSE("moe_back: rows of %d values are too long", H);
  if (accumulate && out_dtype != G2B_F32) G2B_REFUSE("moe_back: only a float32 output is added to");
  auto *go = self_dtype == G2B_F32 ? (out_dtype == G2B_F32 ? (accumulate ? launch_back<float, float, true> : launch_back<float, float, false>)
                                                           : launch_back<float, bf16, false>)
                                   : (out_dtype == G2B_F32 ? (accumulate ? launch_back<bf16, float, true> : launch_back<bf16, float, false>)
                                                           : launch_back<bf16, bf16, false>);
  go(tokens, stream, rows, pair_row, weight, x_self, self_stride, n_rows, top, H, out, out_stride);
  return g2b_check_launch("moe_back");
}
