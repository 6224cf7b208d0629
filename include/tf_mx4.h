/* Microscaled 4-bit weights on gfx950, and the experts' choice that goes with them.
 *
 * A microscaled tensor ("mx4") is the OCP MXFP4 format: along each row, 32 consecutive
 * elements share one e8m0 scale byte s (the value 2^(s - 127), 255: NaN), and an element is
 * an e2m1 code (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two
 * to a byte with the even element in the low half.  Row-major: codes [rows][K / 2], scales
 * [rows][K / 32], K % 32 == 0.  The reference has no 4-bit path; the formulas here are this
 * library's definition.
 *
 * Conventions as in tf_decode.h: device pointers, work enqueued on `stream`, nothing
 * allocated, nothing synchronised, 0 or an error code with tfd_last_error()'s text.  Strides
 * count elements (codes: bytes) between rows.  A call of no rows enqueues nothing. */
#ifndef TF_MX4_H
#define TF_MX4_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types of activations */
#define TFD_TYPE_F32 0
#define TFD_TYPE_BF16 1
#define TFD_TYPE_F16 2

/* Rows to mx4.  For a block with largest magnitude t: e = clamp(floor(log2 t) - 2, -127,
 * 125) (-127 for t = 0), scale byte e + 127, codes round-to-nearest-even of x / 2^e,
 * magnitudes past 6 as 6.  A block with a value that is not finite gets scale byte 255 and
 * zero codes: it stands for NaN.  Up to 2^35 - 2048 values a call (2^35: 64 GiB of bf16);
 * the inverse too.  x: f32, bf16 or f16 [rows][ldx]; any alignment of its
 * element size (16-byte aligned rows are read faster).  codes [rows][ldc], ldc % 4 == 0,
 * 4-byte aligned; scales [rows][lds]. */
int tfd_mx4_quantise(const void* x, int64_t ldx, int type, int64_t rows, int K, void* codes,
                     int64_t ldc, void* scales, int64_t lds, void* stream);
/* The values that codes and scales stand for: exact in f32 and in bf16, up to an infinity
 * where 2^(s - 127) times the code passes the type's range (the scales of tfd_mx4_quantise
 * stay below it); f16 rounds once.  out 4-byte aligned, ldo even. */
int tfd_mx4_dequantise(const void* codes, int64_t ldc, const void* scales, int64_t lds,
                       int64_t rows, int K, void* out, int64_t ldo, int type, void* stream);

/* Weights laid out for the products below, once, at load time: blocks of 16 rows x 128 k
 * (1 KiB; lane l's 16 bytes are the 32 codes of row l % 16 at k 32 (l / 16)), K padded with
 * zeros to a multiple of 128 and N to one of 16; then the scales, 256 bytes for each 16 rows x
 * 512 k.  With codes2 / scales2 (a second matrix of the same shape) the rows alternate, row
 * 2i from the first and 2i + 1 from the second: the experts' (gate, up) pairs; N counts the
 * rows of one matrix.  Contiguous sources, codes 16-byte aligned.  `packed`:
 * tfd_mx4_packed_bytes(N, K) bytes, 2 N rows with a second matrix. */
int64_t tfd_mx4_packed_bytes(int64_t N, int K);
int tfd_mx4_pack(const void* codes, const void* scales, const void* codes2, const void* scales2,
                 int64_t N, int K, void* packed, void* stream);

/* out[m][n] = sum_k x[m][k] W[n][k], f32 sums, each output rounded once to f32 or bf16
 * (out_type).  W packed by tfd_mx4_pack ([N][K], N up to 2^24, K up to 2^22).  x: bf16 [M][ldx], or mx4 with x_scales
 * set (codes [M][ldx bytes], scales [M][ldxs]); rows 16-byte aligned, ldx and ldxs up to
 * 2^23.  The 4-bit counterpart of tfd_gemm_skinny_bf16 / tfd_panel_gemm_bf16 for any M, N
 * and K a multiple of 32, on plain rows.  work (may be NULL): with tfd_mx4_gemm_work_bytes of it, 16-byte
 * aligned and contents free, products of few blocks split K over more of them and add the
 * parts in a second launch, always in the same order; without, the same product in one
 * launch.  One call's at a time. */
typedef struct {
  const void* x;
  int64_t ldx;
  const void* x_scales;
  int64_t ldxs;
  const void* w;
  int M, K, N;
  void* out;
  int64_t ldo;
  int out_type;
  void* work;
  int64_t work_bytes;
} TfdMx4GemmArgs;
/* up to so many rows K is never split: no work */
#define TFD_MX4_WHOLE_ROWS 64
int64_t tfd_mx4_gemm_work_bytes(int M, int K, int N);
/* How a product of these sizes runs on the current device, for tests and measurements: form =
 * rows and columns of a block's outputs, parts of K (with work), and the last blocks that run
 * in quarters.  x_mx4 != 0: microscaled rows. */
int tfd_mx4_gemm_form(int x_mx4, int M, int K, int N, int32_t form[4]);
int tfd_mx4_gemm(const TfdMx4GemmArgs* args, void* stream);

/* The choice of experts after the router's projection.  Replaces the two fixed routers of
 * tfd_route_topk (tf_hybrid.h) where a model scores, biases or groups its experts otherwise.
 *   score   s_e = softmax(l)_e over the row (TFD_SCORE_SOFTMAX) or 1 / (1 + exp(-l_e))
 *           (TFD_SCORE_SIGMOID), in 64 bits: a choice compares values that lie close;
 *   choice  c_e = s_e + bias_e (bias NULL: s_e).  An expert whose logit is NaN or -inf, or
 *           whose bias is NaN or -inf, is never chosen; a logit of +inf shares all of a
 *           softmax with the row's other ones;
 *   groups  experts in `groups` runs of experts / groups; a run ranks by the sum of its best
 *           group_top (1 or 2) choices, and the best kept_groups runs stay;
 *   picks   the k best choices of the runs that stayed, largest first; equal ones (runs too)
 *           by the lower index;
 *   weight  s_e, divided by the picks' sum with renormalise != 0, times scale, in f32.
 * Where fewer than k experts can be chosen the last places hold id -1 and weight 0, and a sum
 * of zero gives weights of zero.  `shared` places follow each row's picks: ids experts,
 * experts + 1, ..., weight 1 (tfd_mx4_experts then adds the shared experts with the rest).
 * logits f32, bf16 or f16 [rows][ldl]; weights f32 and ids int32 [rows][ld], ld >= k + shared.
 * rows <= 67,108,860, experts <= 512, groups <= 64 and a divisor of experts, k + shared <= 64,
 * k <= kept_groups * experts / groups. */
#define TFD_SCORE_SOFTMAX 0
#define TFD_SCORE_SIGMOID 1
#define TFD_ROUTE_MAX_EXPERTS 512
typedef struct {
  const void* logits;
  int64_t ldl;
  int type;
  const float* bias;
  int rows, experts, k, score, groups, kept_groups, group_top, shared, renormalise;
  float scale;
  float* weights;
  int32_t* ids;
  int ld;
} TfdRouteArgs;
int tfd_route_experts(const TfdRouteArgs* args, void* stream);

/* The routed experts over mx4 weights, given the routing: for row r
 *   y = mult * sum over places j of weights[r][j] * Wdown_e (silu(Wgate_e x_r) * (Wup_e x_r)),
 *   e = ids[r][j]; f32 sums; the hidden values (the down product's operands) rounded to bf16,
 *   or in calls of up to 16 rows and 128 places kept as sums of two bf16 (2^-17);
 * out = y, or with accumulate out + y (a residual stream), rounded once to out_type.  Entries
 * are grouped by expert, so a picked expert's weights are read once for all its rows (many
 * rows: once for each 16 to 128).  The 4-bit counterpart of tfd_moe_experts* / tfd_panel_moe;
 * shared experts are experts that every row picks (tfd_route_experts appends them).
 * x bf16 [rows][ldx], rows 16-byte aligned; ids / weights [rows][ld]; w_gu = tfd_mx4_pack of
 * gate [E I][H] with up [E I][H] as its second matrix, w_down of [E H][I]; H and I multiples
 * of 32 up to 2^20, experts <= 512, k <= 64, rows <= 65535, rows * ldx and rows * k * I below 2^30.  Id -1 is an empty place; another id outside
 * the experts is skipped and raises TFD_ERR_TOKEN_RANGE in err (NULL: nothing).  An expert
 * may come twice in a row.  work: tfd_mx4_experts_work_bytes, which never falls as rows grow
 * (one buffer serves its rows and all fewer), 256-byte aligned, contents free, one call's at a
 * time. */
typedef struct {
  const void* x;
  int64_t ldx;
  const int32_t* ids;
  const float* weights;
  int ld;
  const void* w_gu;
  const void* w_down;
  int rows, k, experts, H, I;
  void* out;
  int64_t ldo;
  int out_type, accumulate;
  float mult;
  void* work;
  int64_t work_bytes;
  int32_t* err;
} TfdMx4ExpertsArgs;
int64_t tfd_mx4_experts_work_bytes(int rows, int k, int experts, int H, int I);
/* How a call runs, for tests and measurements: an expert's rows in tiles of up to 16, 64 or
 * 128, or 0 for the two launches of few rows (sizes as tfd_mx4_experts takes them, else -1). */
int tfd_mx4_experts_tile_rows(int rows, int k, int experts, int H, int I);
int tfd_mx4_experts(const TfdMx4ExpertsArgs* args, void* stream);

#ifdef __cplusplus
}
#endif

#endif
