// The operators in 8-bit floating point as they are called: quantisation, products, routed experts.  A call is one function here, whatever it
// launches: on the host a call of its own for every kernel costs more than the kernels of a decode step take.
#include "gemm_fp8_few.cuh"
#include "gemm_fp8_tc.cuh"
#include "quant_fp8.cuh"

G2B_DEFINE_LAST_ERROR

extern "C" int g2b_quantize_rows(const void *x, int dtype, long long x_stride, int tokens, int K, void *q, long long q_stride, float *scale,
                                 long long scale_stride, const int *pair_row, int top, int n_rows, cudaStream_t stream) {
  return run_quantize_rows(x, dtype, x_stride, tokens, K, q, q_stride, scale, scale_stride, pair_row, top, n_rows, stream);
}
extern "C" int g2b_quantize_matrix(const void *w, int dtype, int count, int N, int K, long long w_stride, void *q, long long q_stride, float *scale,
                                   cudaStream_t stream) {
  return run_quantize_matrix(w, dtype, count, N, K, w_stride, q, q_stride, scale, stream);
}
extern "C" int g2b_moe_sort(const int *idx, int n_pairs, int n_real, int *starts, int *pair_row, int *row_pair, cudaStream_t stream) {
  return run_moe_sort(idx, n_pairs, n_real, starts, pair_row, row_pair, stream);
}
extern "C" int g2b_moe_back(const float *rows, const int *pair_row, const float *weight, const void *x_self, int self_dtype, long long self_stride,
                            int n_rows, int tokens, int top, int H, void *out, int out_dtype, long long out_stride, int accumulate, cudaStream_t stream) {
  return run_moe_back(rows, pair_row, weight, x_self, self_dtype, self_stride, n_rows, tokens, top, H, out, out_dtype, out_stride, accumulate, stream);
}

// ---- which kernel ---------------------------------------------------------------------------------------
// columns of gemm_fp8_few.cuh (16, 32, 64, -64; 0: gemm_fp8_tc.cuh), its parts of K, and whether it quantises on the way
struct Choice { int columns, split, with_x; };
enum Way { EITHER_WAY, GIVEN_ROWS, ON_THE_WAY };

// Microseconds that a product is estimated to take.  With `c` CTAs of `n` blocks of K each, as many as `most` at a time:
//   start + (parts + part * split, where K is in parts) + the 4-norm of (the rounds of CTAs: n blocks each, and `wave` for every round but one) and
//   (W's bytes at `rate` TB/s);  a block takes `alone` where no two CTAs share a multiprocessor, else `block`.
// Fitted to 7,000 times of 430 products that are not experts' (1 to 1,500 rows, 256 to 30,000 outputs, K = 512 to 17,408; graphs of products behind one
// another), within 7 to 10 % (root mean square of the logarithm); experts' are taken for as many rows each.  Against the best of all tiles and
// parts that are looked at, with the kernels as they are: 150 products drawn from the same ranges lose 3.6 % in the mean and 25 at worst (73 rows by 14,912 x
// 10,112 44.5 us, 35.6 with 128 rows on the lanes), 80 routed layers (1 to 2,048 tokens, 4 to 122 experts, popular ones among them) 1.0 % and 14.  Not looked at:
// several tiles of rows quantised on the way, 29 rows by 960 x 512 5.4 us for 3.8.  With the tiles the largest that fit instead, 64 rows by 5,120 x 17,408
// took 34 us (21), and 128 rows by 6,144 x 4,096 13.9 (11.1).
struct Cost { double start, parts, part, alone, block, wave, rate; };
constexpr Cost COST_X = {2.11, 0.60, 0.08, 0.348, 0.408, 1.82, 5.75}, COST_16 = {2.02, 0.59, 0.07, 0.238, 0.349, 1.77, 6.42},
               COST_32 = {2.57, 0.58, 0.08, 0.280, 0.411, 2.17, 6.46}, COST_64 = {2.81, 0.55, 0.18, 0.357, 0.550, 2.61, 5.27},
               COST_LANES = {2.89, 0.48, 0.26, 0.271, 0.412, 2.69, 5.67};
constexpr double MANY_START = 2.41, MANY_BLOCK = 0.430, MANY_TILE = 1.88;   // of gemm_fp8_tc.cuh: a round is its blocks and a tile's outputs
constexpr double QUANTISED_FIRST = 2.0, SORTED_FIRST = 2.5;                  // a kernel of its own in front

static double estimate(const Cost &k, long long tiles, int blocks, int split, int most, double w_bytes) {
  const long long ctas = tiles * split, rounds = ctas / most, rest = ctas % most;
  const int n = (blocks + split - 1) / split;
  double work = rounds * (n * k.block + k.wave);
  if (rest) work += n * (rest <= 148 ? k.alone : k.block) + (rounds ? k.wave : 0);
  const double bytes = w_bytes * 1e-6 / k.rate, w2 = work * work, b2 = bytes * bytes;
  return k.start + (split > 1 ? k.parts + k.part * split : 0) + __builtin_sqrt(__builtin_sqrt(w2 * w2 + b2 * b2));
}

// The cheapest for activations that are still to be quantised; given rows go the same way, so that they have the same bits.  `experts`: the rows are
// theirs, as many for each (those that have any), give or take.  rows_needed: quantised rows are to be left (only gemm_fp8_tc.cuh leaves them itself).
static Choice choose(int M, int N, int blocks, int experts, bool rows_needed, Way way = EITHER_WAY, double *estimated = nullptr) {
  const int used = experts ? (experts < M ? experts : M) : 1;
  const long long each = ((long long)M + used - 1) / used;
  const double w_bytes = (double)used * N * blocks * F8_BLOCK;
  const double behind = rows_needed ? QUANTISED_FIRST + 1e-6 * M * N * 2.5 / 4 : 0;      // float, read and written again
  const long long pairs_tiles = used * ((each + 255) / 256) * (((long long)N + 255) / 256);
  const int pairs = many::resident();
  Choice best = {0, 1, 0};
  double least = way == ON_THE_WAY ? INFINITY : QUANTISED_FIRST + MANY_START + (double)((pairs_tiles + pairs - 1) / pairs) * (blocks * MANY_BLOCK + MANY_TILE);
  auto look = [&](int columns, bool x, const Cost &k, int (*resident)(int)) {
    if (way == (x ? GIVEN_ROWS : ON_THE_WAY)) return;
    const int rows_a = columns > 0 ? columns : 128, rows_w = columns > 0 ? 128 : 64;
    const long long tiles_n = ((long long)N + rows_w - 1) / rows_w, tiles = used * ((each + rows_a - 1) / rows_a) * tiles_n;
    if (tiles > INT32_MAX / few::MOST_SPLIT || (!experts && tiles_n > few::MOST_TILES_N)) return;
    for (int split = 1; split <= few::MOST_SPLIT && split <= blocks; ++split) {
      const double us = estimate(k, tiles, blocks, split, resident(split), w_bytes) + (x ? 0 : QUANTISED_FIRST) + behind;
      if (us < least) least = us, best = {columns, split, x};
    }
  };
  if (each <= 16) look(16, true, COST_X, experts ? few::resident<16, false, true, true> : few::resident<16, false, true, false>);
  if (each <= 48) look(16, false, COST_16, experts ? few::resident<16, false, false, true> : few::resident<16, false, false, false>);
  if (each > 8 && each <= 64) look(32, false, COST_32, experts ? few::resident<32, false, false, true> : few::resident<32, false, false, false>);
  if (each > 16 && each <= 128) look(64, false, COST_64, experts ? few::resident<64, false, false, true> : few::resident<64, false, false, false>);
  if (each > 16) look(-64, false, COST_LANES, experts ? few::resident<64, true, false, true> : few::resident<64, true, false, false>);
  if (estimated) *estimated = least;
  return best;
}

static bool on_the_way(const void *x, int x_f32, long long x_stride, int K) {
  return K % 8 == 0 && x_stride % (x_f32 ? 4 : 8) == 0 && ((uintptr_t)x & 15) == 0;
}
static size_t on_16(size_t bytes) { return (bytes + 15) / 16 * 16; }

// What a call's sizes and types fix.
struct Call {
  long long lda, lds, ldw, ldo, ldos, x_stride;
  int M, N, K, x_dtype, epi, n_experts, top, H;          // x_dtype < 0: quantised rows are given
  Choice first, second;                                  // of the product, or the experts' two
  GluForm form;
};
static bool may_be_on_the_way(const Call &c, bool x_aligned) {
  return c.x_dtype >= 0 && x_aligned && on_the_way(nullptr, c.x_dtype == G2B_F32, c.x_stride, c.K);
}

static int check(const Product &p) {
  if (p.ldw % 16 || ((uintptr_t)p.w & 15) || (!p.x && (p.lda % 16 || ((uintptr_t)p.a & 15)))) G2B_REFUSE("products_fp8: rows must start on 16 bytes");
  if (p.gated() && p.N % 16) G2B_REFUSE("products_fp8: gates and ups in eights, got %d rows", p.N);
  if (p.epi == EPI_GATED_ROWS && (p.ldo % 16 || ((uintptr_t)p.out & 15))) G2B_REFUSE("products_fp8: quantised rows must start on 16 bytes");
  if (p.n_experts < 0 || p.n_experts > MOST_EXPERTS || (p.n_experts && !p.starts && !p.idx)) G2B_REFUSE("products_fp8: %d experts outside 1..%d", p.n_experts, MOST_EXPERTS);
  if (p.w_rows() > INT32_MAX || p.lda > INT32_MAX || p.ldw > INT32_MAX) G2B_REFUSE("products_fp8: %lld rows of W are too many", p.w_rows());
  return 0;
}
static int product(const Product &p, Choice c, cudaStream_t stream) {
  const int rc = check(p);
  if (rc) return rc;
  return c.columns ? few::run(p, c.columns, c.split, stream) : many::run(p, stream);
}

// Rows of `k` values, quantised, in scratch memory.
struct Rows {
  uint8_t *q;
  float *scale;
  long long ld, lds;
};
static size_t rows_bytes(long long rows, int k) {
  const size_t blocks = (k + F8_BLOCK - 1) / F8_BLOCK;
  return on_16((size_t)rows * blocks * F8_BLOCK) + on_16((size_t)rows * blocks * 4);
}
static Rows rows_at(unsigned char *&at, long long rows, int k) {
  const long long ld = (k + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK;
  const Rows r = {at, reinterpret_cast<float *>(at + on_16((size_t)rows * ld)), ld, rows};
  at += rows_bytes(rows, k);
  return r;
}
static void take(Product &p, const Rows &r) { p.a = r.q, p.sa = r.scale, p.lda = r.ld, p.lds = r.lds, p.x = nullptr, p.row_pair = nullptr; }

// Gated rows of few rows: the gate in float, then quantised.
static bool by_way_of_float(const Call &c) { return c.epi == EPI_GATED_ROWS && c.first.columns; }

// Chooses the kernel (by_rule: else c->first stands) and returns the bytes of scratch memory that the product takes; x_aligned: x starts on 16 bytes.
extern "C" long long g2b_fp8_product_plan(Call *c, int x_aligned, int by_rule) {
  const bool with_x = may_be_on_the_way(*c, x_aligned != 0);
  if (by_rule) c->first = choose(c->M, c->N, (c->K + F8_BLOCK - 1) / F8_BLOCK, 0, c->epi == EPI_GATED_ROWS);
  if (!with_x) c->first.with_x = 0;
  size_t bytes = 0;
  if (c->x_dtype >= 0 && !c->first.with_x) bytes += rows_bytes(c->M, c->K);
  if (by_way_of_float(*c)) bytes += on_16((size_t)c->M * (c->N / 2) * 4);
  return (long long)bytes;
}

// x: the activations (c->x_dtype), or quantised rows with their scales sa; out_scale: EPI_GATED_ROWS.  Returns how many kernels were launched, or
// less than 0.
extern "C" int g2b_fp8_product(const Call *c, const void *x, const float *sa, unsigned char *scratch, const void *w, const float *sw, void *out,
                               float *out_scale, int *status, cudaStream_t stream) {
  if (c->M <= 0 || c->N <= 0 || c->K <= 0) return 0;
  const Choice choice = c->first;
  Product p = {};
  p.w = w, p.sw = sw, p.out = out, p.out_scale = out_scale, p.status = status;
  p.ldw = c->ldw, p.ldo = c->ldo, p.ldos = c->ldos, p.M = c->M, p.N = c->N, p.K = c->K, p.blocks = (c->K + F8_BLOCK - 1) / F8_BLOCK;
  p.epi = c->epi, p.form = c->form, p.top = 1;
  int launches = 1;
  if (c->x_dtype < 0) {
    p.a = x, p.sa = sa, p.lda = c->lda, p.lds = c->lds;
  } else if (choice.with_x) {
    p.x = x, p.x_f32 = c->x_dtype == G2B_F32, p.x_stride = c->x_stride;
  } else {
    const Rows r = rows_at(scratch, c->M, c->K);
    if (run_quantize_rows(x, c->x_dtype, c->x_stride, c->M, c->K, r.q, r.ld, r.scale, r.lds, nullptr, 1, c->M, stream)) return -1;
    take(p, r);
    ++launches;
  }
  if (!by_way_of_float(*c)) return product(p, choice, stream) ? -1 : launches;
  p.out = scratch, p.ldo = c->N / 2, p.epi = EPI_GATED_F32;
  if (product(p, choice, stream)) return -1;
  if (run_quantize_rows(scratch, G2B_F32, c->N / 2, c->M, c->N / 2, out, c->ldo, out_scale, c->ldos, nullptr, 1, c->M, stream)) return -1;
  return launches + 1;
}

// ---- routed experts -------------------------------------------------------------------------------------
// c: M tokens of K values with `top` choices among n_experts experts of N / 2 outputs between, H behind.  As g2b_fp8_product_plan.
extern "C" long long g2b_fp8_experts_plan(Call *c, int x_aligned, int by_rule) {
  const long long pairs = (long long)c->M * c->top;
  const int inter = c->N / 2, blocks = (c->K + F8_BLOCK - 1) / F8_BLOCK, blocks_down = (inter + F8_BLOCK - 1) / F8_BLOCK;
  size_t bytes = on_16((size_t)(c->n_experts + 1) * 4);
  if (pairs <= 0 || pairs > INT32_MAX) return (long long)bytes;        // (the call has nothing to do, or refuses it)
  if (by_rule) {
    // both products quantise their rows, or neither does; where both do, few pairs need no kernel that sorts them (4 tokens of 6 choices among 64 experts of
    // 768 between 2,048: 22.2 us against 25.0; 16 tokens, sorted first: 52 against 47)
    double us[2][2];
    const Choice given[2] = {choose((int)pairs, c->N, blocks, c->n_experts, true, GIVEN_ROWS, &us[0][0]), choose((int)pairs, c->H, blocks_down, c->n_experts, false, GIVEN_ROWS, &us[0][1])};
    const Choice own[2] = {choose((int)pairs, c->N, blocks, c->n_experts, false, ON_THE_WAY, &us[1][0]), choose((int)pairs, c->H, blocks_down, c->n_experts, false, ON_THE_WAY, &us[1][1])};
    const bool with_x = us[1][0] + us[1][1] - (pairs <= MOST_INLINE ? SORTED_FIRST : 0) < us[0][0] + us[0][1];
    c->first = (with_x ? own : given)[0], c->second = (with_x ? own : given)[1];
  }
  if (!may_be_on_the_way(*c, x_aligned != 0)) c->first.with_x = 0;
  if (!c->first.with_x) c->second.with_x = 0;
  if (c->first.with_x) return (long long)(bytes + on_16((size_t)pairs * 4) + on_16((size_t)pairs * inter * 4));
  bytes += rows_bytes(pairs, c->K) + rows_bytes(pairs, inter);
  if (c->first.columns) bytes += on_16((size_t)pairs * inter * 4);
  return (long long)bytes;
}

// h [M, K] (c->x_dtype), idx [M, top]; w_gu [n_experts, N, ..] gated, w_down [n_experts, H, ..] of N / 2 columns; rows float [M * top, H] in the experts'
// order and pair_row [M * top] are written.  Returns how many kernels were launched, or less than 0.
extern "C" int g2b_fp8_experts(const Call *c, const void *h, const int *idx, unsigned char *scratch, const void *w_gu, const float *s_gu,
                               const void *w_down, const float *s_down, float *rows, int *pair_row, int *status, cudaStream_t stream) {
  if (c->M <= 0 || c->top <= 0) return 0;
  if ((long long)c->M * c->top > INT32_MAX) { snprintf(g2b_error_text, sizeof(g2b_error_text), "fp8_experts: %d tokens are too many", c->M); return -1; }
  const int pairs = c->M * c->top, inter = c->N / 2;
  int *starts = reinterpret_cast<int *>(scratch);
  scratch += on_16((size_t)(c->n_experts + 1) * 4);
  Product p = {};
  p.w = w_gu, p.sw = s_gu, p.status = status, p.starts = starts, p.n_experts = c->n_experts, p.form = c->form, p.top = c->top;
  p.ldw = c->ldw, p.M = pairs, p.N = c->N, p.K = c->K, p.blocks = (c->K + F8_BLOCK - 1) / F8_BLOCK, p.epi = EPI_GATED_F32;
  Product d = p;
  d.w = w_down, d.sw = s_down, d.out = rows, d.ldo = c->H, d.N = c->H, d.K = inter, d.blocks = (inter + F8_BLOCK - 1) / F8_BLOCK, d.ldw = d.blocks * F8_BLOCK;
  d.epi = EPI_F32, d.top = 1;
  const Choice gated = c->first, down = c->second;
  if (c->n_experts < 1) { snprintf(g2b_error_text, sizeof(g2b_error_text), "fp8_experts: %d experts", c->n_experts); return -1; }
  if (gated.with_x) {
    // few rows an expert: their places are enough, the products fetch and quantise them
    int *row_pair = reinterpret_cast<int *>(scratch);
    float *mid = reinterpret_cast<float *>(scratch + on_16((size_t)pairs * 4));
    const bool inline_sort = pairs <= MOST_INLINE;
    p.x = h, p.x_f32 = c->x_dtype == G2B_F32, p.x_stride = c->x_stride, p.out = mid, p.ldo = inter;
    d.x = mid, d.x_f32 = 1, d.x_stride = inter;
    if (inline_sort) {
      p.idx = d.idx = idx, p.starts = d.starts = nullptr, p.pair_row = pair_row, p.gather = 1;
    } else {
      if (run_moe_sort(idx, pairs, c->n_experts, starts, pair_row, row_pair, stream)) return -1;
      p.row_pair = row_pair;
    }
    if (product(p, gated, stream)) return -1;
    return product(d, down, stream) ? -1 : inline_sort ? 2 : 3;
  }
  const Rows sorted = rows_at(scratch, pairs, c->K), between = rows_at(scratch, pairs, inter);
  if (run_moe_sort(idx, pairs, c->n_experts, starts, pair_row, nullptr, stream)) return -1;
  if (run_quantize_rows(h, c->x_dtype, c->x_stride, c->M, c->K, sorted.q, sorted.ld, sorted.scale, sorted.lds, pair_row, c->top, pairs, stream)) return -1;
  take(p, sorted);
  int launches = 4;
  if (gated.columns) {
    p.out = scratch, p.ldo = inter;
    if (product(p, gated, stream)) return -1;
    if (run_quantize_rows(scratch, G2B_F32, inter, pairs, inter, between.q, between.ld, between.scale, between.lds, nullptr, 1, pairs, stream)) return -1;
    ++launches;
  } else {
    p.epi = EPI_GATED_ROWS, p.out = between.q, p.out_scale = between.scale, p.ldo = between.ld, p.ldos = between.lds;
    if (product(p, gated, stream)) return -1;
  }
  take(d, between);
  return product(d, down, stream) ? -1 : launches;
}
