/* step_ops.h -- the operators of a decode step around the cached attention
 * (C ABI): projections with 4-bit weights, the gated feed-forward block on
 * them, and the choice of the next token from penalised, biased and masked
 * logits.
 *
 * The reference keeps fp16 matrices behind ILinearOp (worker/include/ops/
 * op_linear.h) and chooses greedily (op_greedy_sample, worker/src/ops/
 * op_sampling.cpp:4-11); these are the 4-bit form of the one and the
 * controls of the other.  qwen2_engine.h runs a whole model on them
 * (qw2_quantize_weights, qw2_set_controls).
 *
 * Conventions are those of kvattn.h: int status, kv_last_error(), device
 * pointers, `stream` a cudaStream_t as void*.  The calls allocate nothing and
 * keep nothing between calls, so they may be captured into a CUDA graph and may
 * run on several streams at once (with scratch of their own, where they take it).  `device` says
 * where the pointers live; the calling thread's current device is kept.
 */
#ifndef STEP_OPS_H
#define STEP_OPS_H

#include <stddef.h>
#include <stdint.h>

#include "kvattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of activations, logits and weights to quantise (the values
 * of QW2_F16, QW2_BF16 and QW2_F32). */
enum { STEP_F16 = 0, STEP_BF16 = 1, STEP_F32 = 2 };

/* A matrix W [n][k] (n outputs, k inputs) in 4 bits: weight (r, i) is
 *   (code(r, i) - zero(r, i / group)) * scale(r, i / group),
 * codes 0..15, zero points 0..15 (8 everywhere where `zeros` is NULL),
 * fp16 scales; group is 32, 64 or 128, the last group of a row may be short.
 *
 * Layout, in tiles of 16 rows and spans of 128 inputs (T = ceil(n / 16),
 * S = ceil(k / 128), Q = ceil(k / group)):
 *   codes   uint32 [T][S][2][32][4]: word [t][s][h][4 g + c][j] holds row
 *           16 t + 8 h + g, inputs 128 s + 32 j + 8 c + i, i = 0..7, input i
 *           in the four bits from 4 * {0, 4, 1, 5, 2, 6, 3, 7}[i]: one warp
 *           reads a tile's span (1 KiB) with two 16-byte loads per lane, and
 *           the words unpack into the operands of its matrix instructions
 *           in input order;
 *   scales  fp16 [T][Q][8][2]: element [t][q][g][h] is row 16 t + 8 h + g;
 *   zeros   uint8, the same shape, or NULL.
 * Codes and scales of the last tile's and span's padding have to be there
 * (they are read) and may hold anything.  All three are 16-byte aligned. */
typedef struct w4_matrix {
    int device;
    int n, k, group;
    void* codes;
    void* scales;
    void* zeros;
} w4_matrix;

/* Bytes of the three arrays of an n x k matrix. */
int w4_sizes(int n, int k, int group, size_t* codes, size_t* scales, size_t* zeros);

/* Bring W [n][k] (STEP_F16 or STEP_BF16, rows ldw elements apart) to 4 bits in
 * m's arrays.  Every step is one IEEE fp32 operation or rounding, so the
 * codes are the same everywhere.  Without zero points (m->zeros NULL):
 * scale = fp16(max|w| / 7), code = clamp(rint(w / scale) + 8, 0, 15).  With
 * them: lo = min(w, 0), hi = max(w, 0) over the group, scale = fp16((hi - lo)
 * / 15), zero = clamp(rint(-lo / scale), 0, 15), code = clamp(rint(w /
 * scale) + zero, 0, 15).  A group whose scale is 0 (all zeros, or all below
 * fp16's range) gets code = zero = 8.  Weights have to be finite and a
 * group's scale within fp16's range. */
int w4_quantize(const w4_matrix* m, const void* w, int dtype, long long ldw, void* stream);

/* The values of m as fp32 rows, ldo elements apart. */
int w4_dequantize(const w4_matrix* m, float* out, long long ldo, void* stream);

/* out[r][i] = sum_k x[r][k] W[i][k] (+ bias[i]) (+ residual[r][i]) for m rows,
 * m >= 0.  x: x_dtype, rows ldx elements apart; out and residual: out_dtype,
 * rows ldo and ldr apart; bias fp32 or NULL; residual may be NULL, or out
 * itself.  Sums are fp32; an fp32 x keeps all its bits (three bf16 parts);
 * the result is rounded once.  A group's sum of (code - zero) * x is formed
 * before its scale, so that sum has to stay within fp32 (|x| below 1e35 does).
 * out must not overlap x; they may be columns of one buffer (rows the same
 * distance apart in bytes: otherwise spans that meet are refused).  The same
 * holds for residual and out, and for the rows of logits_adjust.
 * work: w4_work_bytes() of scratch, 16-byte aligned, overlapping nothing else,
 * or NULL: many rows of an x that is fp32, or not in 16-byte aligned rows, go
 * through it, and take longer without it. */
int w4_linear(const w4_matrix* w, const void* x, int x_dtype, int m, long long ldx, const float* bias,
              const void* residual, long long ldr, void* out, int out_dtype, long long ldo, void* work, void* stream);

/* out = silu(x Wg^T) * (x Wu^T), silu(a) = a / (1 + exp(-a)): the first half
 * of a gated feed-forward block.  gate and up have the same n, k, group and
 * device, and both or neither have zero points. */
int w4_gated(const w4_matrix* gate, const w4_matrix* up, const void* x, int x_dtype, int m, long long ldx, void* out,
             int out_dtype, long long ldo, void* work, void* stream);

/* Scratch of w4_linear (gated 0) or w4_gated (gated 1) for m rows of x: 0
 * where none helps. */
int w4_work_bytes(int n, int k, int group, int x_dtype, int m, int gated, size_t* bytes);

/* The waits inside the kernels for many rows are bounded (about a second):
 * *status is KV_OK, or KV_ERR_TIMEOUT if one has run out in a call on `device`
 * since the last step_ops_status (what that call's out holds is then
 * unspecified: some of it may be written, some of that from unfinished sums).
 * Synchronises the device.  A model's forwards report their own (KV_ERR_TIMEOUT
 * from the forward), and not here. */
int step_ops_status(int device, int* status);

/* The limit of those waits, in SM clocks, for every launch of this process from
 * now on: 0 gives up wherever something is not ready yet, < 0 is the default. */
int step_ops_wait_limit(long long clocks);

/* Penalties, biases, a mask and the greedy choice on `rows` rows of logits.
 * For row r and token t, in fp32, each step rounded by itself:
 *   l = logits[r][t]
 *   if t is in the row's history:        l = l > 0 ? l / repetition : l * repetition
 *   if t is in its generated part:       l = l - frequency * count, then l = l - presence
 *   if t is in the row's bias list:      l = l + the value of its last entry there
 *   if the mask forbids t:               l = -inf, whatever the logit was (NaN too)
 *   out[r][t] = l in dtype
 * and pick[r] = the lowest t with the largest l above -FLT_MAX (NaN never
 * counts; the order of op_greedy_sample), -1 where there is none, as where a
 * mask leaves nothing.  The choice is made on the fp32 values.
 *
 * History: the ids hist[hist_off[r]] .. hist[hist_off[r + 1] - 1]; those from
 * gen_from[r] on (counted from the row's first) are its generated part, the
 * whole history where gen_from is NULL.  Ids outside [0, vocab) count for nothing.
 * Bias lists: bias_ids / bias, cut by bias_off the same way.  Offsets are
 * held within [0, hist_n] and [0, bias_n].  mask: bit t % 32 of word t / 32
 * of the row's ld_mask words, 1 = allowed; bits from vocab on are not read
 * as tokens.  hist, bias_ids, mask, pick and the penalties may be NULL (none;
 * repetition 1).  out may be logits itself (same ld); another overlap is
 * refused.  Rows of out that start at another distance from a 16-byte boundary
 * than those of logits are written value by value, which takes longer. */
typedef struct logits_call {
    int device, rows, vocab, dtype;
    const void* logits;
    long long ld_logits;
    void* out;
    long long ld_out;
    int* pick;                /* [rows] or NULL */
    const int* hist;
    const int* hist_off;      /* [rows + 1] */
    const int* gen_from;      /* [rows] or NULL */
    long long hist_n;         /* ids in hist */
    const float* repetition;  /* [rows] each, or NULL */
    const float* presence;
    const float* frequency;
    const int* bias_ids;
    const float* bias;
    const int* bias_off;      /* [rows + 1] */
    long long bias_n;
    const uint32_t* mask;
    long long ld_mask;        /* words from row to row */
} logits_call;

int logits_adjust(const logits_call* call, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* STEP_OPS_H */
