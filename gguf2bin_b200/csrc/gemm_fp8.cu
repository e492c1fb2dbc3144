// Products in 8-bit floating point (fp8.cuh):  C[t, n] = sum_b s[b, t] S[n / 128, b] sum_{k in block b} q[t, k] Q[n, k].
//
// A tile of 64 rows of A and 64 of W a block of threads, four warps of 32 x 32 on mma.m16n8k32.  The sums of a block of 128 of K come from the
// tensor cores; times the two scales they are added to sums in registers.  `starts`: W is a stack of matrices and rows starts[e] .. starts[e + 1] of
// A meet the e-th.  Gated: rows of W alternate, eight gates and the eight ups of the same outputs, each with the scales of their own matrix.
#include "fp8.cuh"
#include "glu.cuh"

G2B_DEFINE_LAST_ERROR

enum { EPI_BF16 = 0, EPI_F32 = 1, EPI_ADD_F32 = 2, EPI_GATED_F32 = 3 };

struct Product {
  const uint8_t *a, *w;
  const float *sa, *sw;
  void *out;
  const int *starts;
  int M, N, blocks, n_experts;
  long long lda, ldw, lds, ldo;
  GluForm form;
};

constexpr int T_M = 64, T_N = 64, PITCH = F8_BLOCK + 16;

template <int EPI>
__global__ void __launch_bounds__(128)
gemm_fp8_kernel(const Product p) {
  __shared__ __align__(16) uint8_t sh[2][T_M][PITCH];
  __shared__ int found[3];
  pdl_launch();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  int m0 = blockIdx.y * T_M, end = p.M, e = 0;
  if (p.starts) {
    if (threadIdx.x == 0) {
      int left = blockIdx.y, at = 0;
      for (; at < p.n_experts; ++at) {
        const int tiles = (p.starts[at + 1] - p.starts[at] + T_M - 1) / T_M;
        if (left < tiles) break;
        left -= tiles;
      }
      found[0] = at;
      found[1] = at < p.n_experts ? p.starts[at] + left * T_M : 0;
      found[2] = at < p.n_experts ? p.starts[at + 1] : 0;
    }
    __syncthreads();
    e = found[0], m0 = found[1], end = found[2];
    if (e >= p.n_experts) return;
  }
  const int n0 = blockIdx.x * T_N;
  constexpr bool GATED = EPI == EPI_GATED_F32;
  const int nb_all = ((GATED ? p.N / 2 : p.N) + F8_BLOCK - 1) / F8_BLOCK;
  const uint8_t *w = p.w + (long long)e * p.N * p.ldw;
  const float *sw = p.sw + ((long long)e * (GATED ? 2 : 1) * nb_all + (GATED ? n0 / 2 : n0) / F8_BLOCK) * p.blocks;
  const long long up = (long long)nb_all * p.blocks;
  const int wm = (warp >> 1) * 32, wn = (warp & 1) * 32;
  float acc[2][4][4] = {};
  for (int b = 0; b < p.blocks; ++b) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * T_M * 8; i += 128) {
      const int which = i / (T_M * 8), r = i / 8 % T_M, at = 16 * (i % 8);
      const int row = which ? n0 + r : m0 + r;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < (which ? p.N : end)) v = *reinterpret_cast<const uint4 *>((which ? w + row * p.ldw : p.a + row * p.lda) + b * F8_BLOCK + at);
      *reinterpret_cast<uint4 *>(&sh[which][r][at]) = v;
    }
    __syncthreads();
    float part[2][4][4] = {};
#pragma unroll
    for (int k = 0; k < F8_BLOCK; k += 32) {
      uint32_t a[2][4], w2[4][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) a[i][r] = *reinterpret_cast<const uint32_t *>(&sh[0][wm + 16 * i + g + 8 * (r & 1)][k + 4 * c + 16 * (r >> 1)]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) w2[j][r] = *reinterpret_cast<const uint32_t *>(&sh[1][wn + 8 * j + g][k + 4 * c + 16 * r]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) mma_e4m3_16832(part[i][j], a[i][0], a[i][1], a[i][2], a[i][3], w2[j][0], w2[j][1]);
    }
    const float s0 = sw[b], s1 = GATED ? sw[up + b] : s0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = m0 + wm + 16 * i + g + 8 * h;
        const float sa = row < end ? p.sa[b * p.lds + row] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float f = sa * (j & 1 ? s1 : s0);
          acc[i][j][2 * h] = fmaf(part[i][j][2 * h], f, acc[i][j][2 * h]);
          acc[i][j][2 * h + 1] = fmaf(part[i][j][2 * h + 1], f, acc[i][j][2 * h + 1]);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long row = m0 + wm + 16 * i + g + 8 * h;
      if (row >= end) continue;
#pragma unroll
      for (int j = 0; j < 4; j += GATED ? 2 : 1)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int n = n0 + wn + 8 * j + 2 * c + x;
          if (n >= p.N) continue;
          const float v = acc[i][j][2 * h + x];
          if (GATED) {
            const int out = (n >> 4) * 8 + (n & 7);
            static_cast<float *>(p.out)[row * p.ldo + out] = glu_value(v, acc[i][j + 1][2 * h + x], p.form);
          } else if (EPI == EPI_BF16) {
            static_cast<bf16 *>(p.out)[row * p.ldo + n] = __float2bfloat16_rn(v);
          } else {
            float *to = static_cast<float *>(p.out) + row * p.ldo + n;
            *to = EPI == EPI_ADD_F32 ? *to + v : v;
          }
        }
    }
}

// a [M, lda], w [N, ldw] (`starts`: [n_experts, N, ldw]), scales sa [blocks, lds] and sw [ceil(N / 128), blocks] (gated: [2, ceil(N / 256), blocks]; a
// stack: for every expert).  Rows of a and w on 16 bytes, zeros behind K.
extern "C" int g2b_gemm_fp8(const void *a, const float *sa, const void *w, const float *sw, void *out, int M, int N, int blocks, long long lda,
                            long long lds, long long ldw, long long ldo, int epi, float limit, float offset, float c1, float c3, const int *starts,
                            int n_experts, cudaStream_t stream) {
  if (M <= 0 || N <= 0 || blocks <= 0) return 0;
  if (lda % 16 || ldw % 16 || (((uintptr_t)a | (uintptr_t)w) & 15)) G2B_REFUSE("gemm_fp8: rows must start on 16 bytes");
  if (epi == EPI_GATED_F32 && N % 16) G2B_REFUSE("gemm_fp8: gates and ups in eights, got %d rows", N);
  Product p;
  p.a = (const uint8_t *)a, p.w = (const uint8_t *)w, p.sa = sa, p.sw = sw, p.out = out, p.starts = starts;
  p.M = M, p.N = N, p.blocks = blocks, p.n_experts = n_experts;
  p.lda = lda, p.ldw = ldw, p.lds = lds, p.ldo = ldo;
  p.form.limit = limit, p.form.offset = offset, p.form.c1 = c1, p.form.c3 = c3;
  const long long tiles_m = ((long long)M + T_M - 1) / T_M + (starts ? n_experts : 0);
  if (tiles_m > 65535) G2B_REFUSE("gemm_fp8: %d rows are too many for one launch", M);
  const dim3 grid((unsigned)((N + T_N - 1) / T_N), (unsigned)tiles_m);
  auto *kernel = epi == EPI_BF16 ? gemm_fp8_kernel<EPI_BF16> : epi == EPI_F32 ? gemm_fp8_kernel<EPI_F32>
                 : epi == EPI_ADD_F32 ? gemm_fp8_kernel<EPI_ADD_F32> : gemm_fp8_kernel<EPI_GATED_F32>;
  g2b_launch(kernel, grid, dim3(128), 0, stream, p);
  return g2b_check_launch("gemm_fp8");
}
