/* c4s_layers.h -- C ABI of the decoder layer's operators (libc4s_sampling.so):
 * what gives the hidden rows that c4s_lmhead_sample turns into tokens.
 *
 * One decoder layer, over a prompt or over one new token a sequence:
 *
 *   c4s_block_norm   the block's output joins the residual stream, the norm in front of the next block
 *   c4s_linear       queries, keys and values (bias)
 *   c4s_kv_append    keys and values into the paged cache, as bf16 or 8-bit codes
 *   c4s_attn         the new tokens over the cache
 *   c4s_linear       onto the residual stream (bias, residual); into the MLP (bias, activation); out of it
 *
 * The reference does this step with MLX (src/t2s/gpt2.cpp); nothing here
 * replaces one of its functions.
 *
 * Conventions are those of c4s_sampling.h: status codes, device pointers, work
 * queued on the given stream, text of the last failure from c4s_last_error. A
 * call that fails its checks queues nothing. A call with no rows queues nothing
 * and returns C4S_OK. All of them may be captured into a graph (c4s_attn and
 * c4s_linear with a workspace: after a call of that size outside a capture).
 * Graphs captured on one stream share those calls' workspace, so their replays
 * must not overlap, as c4s_sampling.h says of its own; here an overlap also
 * leaves counters in the workspace off zero, and later replays are wrong too.
 *
 * Activations are bf16, the residual stream bf16 or fp32; sums, softmax
 * statistics and norms are fp32. Row strides are in elements.
 */
#ifndef C4S_LAYERS_H
#define C4S_LAYERS_H

#include <stdint.h>

#include "c4s_sampling.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms around a block ---------------------------------------------------------
 *
 *   r     = x + res_scale * gate (.) u        u = y, or post_norm(y)
 *   x_out = r
 *   out   = norm(r)                           of r before x_out's rounding
 *   norm(v) = (v - mean) / sqrt(var + eps) * gamma + beta       C4S_NORM_LAYER (biased variance, nn.cpp:73-83)
 *           = v / sqrt(mean(v^2) + eps) * gamma + beta          C4S_NORM_RMS
 *
 * Without y (NULL) r is x. x_out may be x itself. */
enum { C4S_NORM_LAYER = 0, C4S_NORM_RMS = 1 };

typedef struct c4s_norm {
  int32_t M, D;             /* rows; D in 1 .. 16384 */
  int32_t kind;             /* C4S_NORM_* */
  float eps;
  const void* x;            /* [M][ldx] in x_dtype (C4S_DTYPE_*) */
  int64_t ldx;
  int32_t x_dtype;
  int32_t y_dtype;
  const void* y;            /* [M][ldy] in y_dtype, or NULL */
  int64_t ldy;
  int32_t post;             /* 1: u = norm(y) with post_gamma, post_beta; 0: u = y */
  int32_t gate_rows;        /* rows that share one row of gate, >= 1: row m's is gate[m / gate_rows] */
  const float* post_gamma;  /* [D] or NULL (= 1) */
  const float* post_beta;   /* [D] or NULL (= 0) */
  const float* gate;        /* [ceil(M / gate_rows)][ld_gate] or NULL (= 1) */
  int64_t ld_gate;
  float res_scale;
  int32_t out_dtype;
  const float* gamma;       /* [D] or NULL (= 1) */
  const float* beta;        /* [D] or NULL (= 0) */
  void* x_out;              /* [M][ld_x_out] in x_dtype, or NULL */
  int64_t ld_x_out;
  void* out;                /* [M][ld_out] in out_dtype, or NULL */
  int64_t ld_out;
} c4s_norm;

int c4s_block_norm(c4s_ctx* ctx, const c4s_norm* norm, void* stream);

/* ---- linear -------------------------------------------------------------------------
 *
 *   out[m][n] = residual[m][n] + act(sum_k x[m][k] w[n][k] + bias[n])
 *
 * weight is stored (out, in) as nn.cpp:11-16 has it: bf16, or 8-bit codes with
 * w[n][k] = wscale[n][k / group] q[n][k] + wbias[n][k / group] (C4S_W_Q8, as in
 * c4s_head; a row of x with an infinite value gives NaN there, since codes and
 * offsets are summed apart). C4S_ACT_GELU is the tanh form, y/2 (1 + tanh(sqrt(2/pi) (y + 0.044715 y^3))). out may
 * be residual itself when both have one type and stride.
 * K must be a multiple of 8, and of group for 8-bit codes; x, weight and ldx
 * such that every row starts on 16 bytes (8-bit codes: 8); else C4S_EINVAL. */
enum { C4S_ACT_NONE = 0, C4S_ACT_GELU = 1, C4S_ACT_SILU = 2, C4S_ACT_RELU = 3 };

typedef struct c4s_linear_desc {
  int32_t M, N, K;          /* M up to 1073741824, N and K up to 4194304; ceil(M / 128) * ceil(N / 128) up to 16777208 */
  int32_t act;              /* C4S_ACT_* */
  const uint16_t* x;        /* [M][ldx] bf16 */
  int64_t ldx;              /* up to 4194304 */
  const void* weight;       /* [N][K] in wdtype */
  int32_t wdtype;           /* C4S_W_BF16 or C4S_W_Q8 */
  int32_t group;            /* C4S_W_Q8: 32, 64 or 128 */
  const float* wscale;      /* C4S_W_Q8: [N][K / group] */
  const float* wbias;
  const float* bias;        /* [N] or NULL */
  const void* residual;     /* [M][ld_res] in res_dtype, or NULL */
  int64_t ld_res;
  int32_t res_dtype;
  int32_t out_dtype;
  void* out;                /* [M][ld_out] in out_dtype */
  int64_t ld_out;
} c4s_linear_desc;

int c4s_linear(c4s_ctx* ctx, const c4s_linear_desc* lin, void* stream);

/* ---- the paged cache ------------------------------------------------------------------
 *
 * A page holds page_size consecutive positions of one sequence, head by head:
 *   k        [n_pages][n_kv_heads][page_size][head_dim]
 *   v        [n_pages][n_kv_heads][head_dim][page_size]
 * bf16, or (C4S_KV_Q8) int8 codes with one fp32 scale a position and head,
 *   k_scale, v_scale  [n_pages][n_kv_heads][page_size],
 * of which code * scale is the value: scale = max |row| / 127, code =
 * round to even(value / scale); a row of zeros has scale 0. A row with a value
 * that is not finite reads back as NaN.
 * (The values lie with their positions next to each other because that is how
 * the product of weights and values reads them: no transpose in the decode.)
 *
 * block_table[b][i] is the page of sequence b's positions i * page_size and on.
 * An entry outside [0, n_pages) is a page that is not there: nothing is written
 * to it, nothing in it is seen by c4s_attn, and it reads back as zeros. The same
 * holds for positions from max_pages * page_size on.
 *
 * Calls pass the tokens of several sequences packed: rows_off[b] .. rows_off[b+1]
 * are the rows of sequence b's last tokens, the positions lens[b] - n .. lens[b] - 1
 * with n the number of rows (rows_off NULL: one row a sequence, row b). lens
 * counts the new tokens. */
enum { C4S_KV_BF16 = 0, C4S_KV_Q8 = 1 };

typedef struct c4s_kv_cache {
  void* k;
  void* v;                      /* both 16-byte aligned */
  float* k_scale;               /* C4S_KV_Q8, 16-byte aligned */
  float* v_scale;
  const int32_t* block_table;   /* [n_seqs][table_ld] */
  int64_t table_ld;
  int32_t n_seqs;               /* up to 65535 */
  int32_t max_pages;            /* entries of a row of block_table in use, <= table_ld; max_pages * page_size up to 2097152 */
  int32_t n_pages;
  int32_t page_size;            /* 16, 32, 64, 128 or 256 */
  int32_t n_kv_heads;           /* n_kv_heads * page_size * head_dim up to 536870912 */
  int32_t head_dim;             /* a multiple of 16, 16 .. 256 */
  int32_t store;                /* C4S_KV_* */
} c4s_kv_cache;

/* Rows of keys and values: row r's head h at k + r * ldk + h * head_dim. */
typedef struct c4s_kv_rows {
  void* k;                      /* [n_rows][ldk], 8-byte aligned, ldk a multiple of 4 */
  void* v;
  int64_t ldk, ldv;
  const int32_t* lens;          /* [n_seqs] */
  const int32_t* rows_off;      /* [n_seqs + 1] or NULL */
  int32_t n_rows;               /* n_rows * n_kv_heads up to 536870912 */
  int32_t dtype;                /* c4s_kv_append: C4S_DTYPE_BF16; c4s_kv_read: or C4S_DTYPE_F32 */
} c4s_kv_rows;

/* Writes the rows into the cache at their positions. */
int c4s_kv_append(c4s_ctx* ctx, const c4s_kv_cache* cache, const c4s_kv_rows* rows, void* stream);
/* The cache's values at the rows' positions, into the rows. */
int c4s_kv_read(c4s_ctx* ctx, const c4s_kv_cache* cache, const c4s_kv_rows* rows, void* stream);

/* ---- attention over the paged cache --------------------------------------------------
 *
 * Row r of head h, at position p of its sequence, sees the positions j with
 * first[b] <= j <= p that have a page:
 *   out[r][h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q[r][h] . k_j),
 * with the keys and values of head h / (n_heads / n_kv_heads); a row that sees
 * nothing is zero. Values that are not finite matter only to rows that see them
 * (those read inf or NaN).
 * Refused (C4S_EINVAL): max_pages above 1024 together with more than 262144 of
 * (sequence, key head, 16 of its new rows' query heads), where few rows a sequence
 * have their positions' parts joined, or with more than 16777215 of (such a one of
 * a single sequence, part of its positions), of which there are up to 128 parts. */
typedef struct c4s_attn_desc {
  const uint16_t* q;            /* [n_rows][ldq] bf16: row r's head h at q + r * ldq + h * head_dim; 16-byte aligned, ldq a multiple of 8 */
  int64_t ldq;
  uint16_t* out;                /* [n_rows][ld_out] bf16; 8-byte aligned, ld_out a multiple of 4 */
  int64_t ld_out;
  float* lse;                   /* [n_rows][n_heads] log sum_j w_j (-inf where nothing is seen), or NULL */
  const int32_t* lens;          /* [n_seqs] */
  const int32_t* rows_off;      /* [n_seqs + 1] or NULL (one row a sequence) */
  const int32_t* first;         /* [n_seqs] or NULL (= 0): the positions before it are padding */
  int32_t n_rows;
  int32_t max_new;              /* with rows_off: rows a sequence has at most; what is beyond is not computed. Without it not
                                   looked at (a sequence has one row). min(max_new, n_rows) * n_heads up to 536870912 */
  int32_t n_heads;              /* a multiple of the cache's n_kv_heads */
  float scale;
} c4s_attn_desc;

int c4s_attn(c4s_ctx* ctx, const c4s_kv_cache* cache, const c4s_attn_desc* attn, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* C4S_LAYERS_H */
