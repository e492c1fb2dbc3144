// What the kernels of products in 8-bit floating point (gemm_fp8_few.cuh, gemm_fp8_tc.cuh) are given.
#pragma once
#include "fp8.cuh"
#include "glu.cuh"
#include "tc_common.cuh"

using namespace tc;

// stored in bfloat16, in float, added to float; the gate of two products in float, or as the quantised rows of the product behind it
enum { EPI_BF16 = 0, EPI_F32 = 1, EPI_ADD_F32 = 2, EPI_GATED_F32 = 3, EPI_GATED_ROWS = 4 };

constexpr int MOST_INLINE = 32;

// C[t, n] = sum_b s[b, t] S[n / 128, b] sum_{k in block b} q[t, k] Q[n, k]:  a = q [M, lda] with sa = s [blocks, lds], or, in place of both, the
// activations x themselves; w = Q [N, ldw] with sw = S [ceil(N / 128), blocks] (gated: gate and up rows in eights in turn, [2, ceil(N / 256), blocks]).
// Rows of a and w on 16 bytes, zeros behind K.
// n_experts > 0: w is a stack of as many matrices (and sw of their scales), and rows starts[e] .. starts[e + 1] meet the e-th.  Or, with idx in place of
// starts, x in place of a and M <= MOST_INLINE: the rows are sorted by the kernel itself, pair r of M being the idx[r]-th expert's (see moe_sort).
struct Product {
  const void *a, *w;
  const float *sa, *sw;
  void *out;                                             // [M, ldo]
  float *out_scale;                                      // EPI_GATED_ROWS: [blocks of the outputs, ldos]
  const int *starts, *idx;
  int *pair_row;                                         // with idx: where every pair's row is left, or null
  int *status;                                           // where a wait that gives up leaves its code
  const void *x;                                         // [.., K], rows x_stride apart; row r of the product is x's row r, or, with
  const int *row_pair;                                   // row_pair, row_pair[r] / top; with idx and gather, the row's pair / top
  long long lda, ldw, lds, ldo, ldos, x_stride;
  int M, N, K, blocks, n_experts, epi, x_f32, top, gather;
  GluForm form;

  bool gated() const { return epi == EPI_GATED_F32 || epi == EPI_GATED_ROWS; }
  int scale_rows() const { return ((gated() ? N / 2 : N) + F8_BLOCK - 1) / F8_BLOCK; }
  long long w_rows() const { return (long long)N * (n_experts ? n_experts : 1); }
};

#define F8_RW8(r, o) "+r"(r[o]), "+r"(r[o + 1]), "+r"(r[o + 2]), "+r"(r[o + 3]), "+r"(r[o + 4]), "+r"(r[o + 5]), "+r"(r[o + 6]), "+r"(r[o + 7])
