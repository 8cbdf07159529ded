/* c4s_batch.h -- C ABI of what a batch of sequences over the paged cache needs
 * beside the layer's operators (libc4s_sampling.so):
 *
 *   c4s_rope         queries and keys turned by their positions' angles, before c4s_kv_append and c4s_attn
 *   c4s_pages_grow   pages for the sequences' next tokens; the new rows' offsets, positions and slots
 *   c4s_pages_trim   tokens taken back, their pages free again
 *   c4s_pages_fork   beams take over each other's pages
 *   c4s_kv_copy      shared pages copied before they are written
 *   c4s_beam_step    the best continuations of every group of beams, their states in the new order
 *
 * The reference has none of them (its GPT-2 has learned positions, its batch one
 * sequence a row); they stand beside c4s_layers.h and c4s_sampling.h, whose
 * conventions hold: status codes, device pointers, work queued on the given
 * stream, text of the last failure from c4s_last_error; a call that fails its
 * checks queues nothing, one without rows queues nothing and returns C4S_OK.
 * All may be captured into a graph (c4s_beam_step, which has a workspace, after
 * a call of that size outside a capture, and with c4s_layers.h's rule on
 * replays of graphs captured on one stream).
 */
#ifndef C4S_BATCH_H
#define C4S_BATCH_H

#include <stdint.h>

#include "c4s_layers.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rotary positions ---------------------------------------------------------------
 *
 * The first rot_dim dims of a head are rot_dim / 2 pairs (a, b); pair i of a row at
 * position p is turned by the angle t = p * freq[i], and scaled:
 *   a' = scale (a cos t - b sin t),  b' = scale (a sin t + b cos t)
 * C4S_ROPE_HALF: pair i is dims i and i + rot_dim / 2; C4S_ROPE_PAIRS: dims 2 i and
 * 2 i + 1. The other dims are copied. freq is in 64 bits, and angles are reduced to a
 * part of a turn with what their products lose, so that 2^-26 of a turn is all they are
 * off by at every position (a frequency below 1 that is rounded to 32 bits is off by up to
 * 0.03 radians at position 10^6). Negated frequencies turn back.
 * (Contexts longer than a model was trained with: freq and scale as it wants them.)
 *
 * q and k have n_rows rows, row r's head h at q + r * ldq + h * head_dim (strides in
 * elements); the outputs may be the inputs themselves, with the same stride, and
 * must not overlap them otherwise. Positions are pos[r], or, without pos, those of
 * c4s_kv_rows: rows_off[b] .. rows_off[b + 1] are the last positions of lens[b]
 * (rows_off NULL: row b is position lens[b] - 1). Rows of no sequence and positions
 * below 0 are left alone. */
enum { C4S_ROPE_HALF = 0, C4S_ROPE_PAIRS = 1 };

typedef struct c4s_rope_desc {
  const void* q;             /* in dtype, or NULL */
  void* q_out;
  const void* k;             /* in dtype, or NULL */
  void* k_out;
  int64_t ldq, ldq_out, ldk, ldk_out;
  const double* freq;        /* [rot_dim / 2], radians a position */
  const int32_t* pos;        /* [n_rows], or NULL */
  const int32_t* lens;       /* [n_seqs], without pos */
  const int32_t* rows_off;   /* [n_seqs + 1] or NULL */
  int32_t n_seqs;            /* up to 65535 */
  int32_t n_rows;            /* up to 16777215 */
  int32_t n_heads;           /* of q; 1 .. 65535 each where there is a tensor */
  int32_t n_kv_heads;        /* of k */
  int32_t head_dim;          /* 2 .. 1024 */
  int32_t rot_dim;           /* even, 2 .. head_dim */
  int32_t layout;            /* C4S_ROPE_* */
  int32_t dtype;             /* C4S_DTYPE_BF16 or C4S_DTYPE_F32 */
  float scale;
} c4s_rope_desc;

int c4s_rope(c4s_ctx* ctx, const c4s_rope_desc* rope, void* stream);

/* ---- pages handed out -----------------------------------------------------------------
 *
 * The caller's device memory that says which sequence has which pages; the layers'
 * caches (c4s_kv_cache) share block_table. A batch begins with every entry of
 * block_table -1, lens and refs 0, and every page's bit of free_bits set.
 * A sequence's row of block_table holds the pages of its lens tokens, and -1 behind
 * them. refs[p] is the number of sequences whose table holds page p, free_bits says
 * the same as refs[p] == 0; bits behind the last page are clear. A program may hold
 * pages of its own (a prompt's beginning that is kept) by a count and a clear bit.
 * Entries of block_table outside [0, n_pages) are no pages.
 *
 * Calls are made on one stream, or ordered by the caller: each reads what the last
 * one wrote. */
typedef struct c4s_pages {
  int32_t* block_table;      /* [n_seqs][table_ld] */
  int64_t table_ld;
  int32_t* lens;             /* [n_seqs] */
  int32_t* refs;             /* [n_pages] */
  uint32_t* free_bits;       /* [ceil(n_pages / 32)]: bit p % 32 of word p / 32; 16-byte aligned */
  int32_t* missing;          /* [1], or NULL: pages that were asked for in vain are added to it */
  int32_t n_seqs;            /* up to 4096 */
  int32_t max_pages;         /* entries of a row in use, <= table_ld; max_pages * page_size up to 2097152 */
  int32_t n_pages;           /* n_pages * page_size up to 2147483647 */
  int32_t page_size;         /* 16, 32, 64, 128 or 256 */
} c4s_pages;

/* lens[b] += n_new[b] (below 0: 0; all of them together, and every length, stay below
 * 2^31), with the pages for it: the free ones with the lowest numbers, to the sequences
 * in order. What is not to be had, or lies behind
 * max_pages, is counted in missing; its entries stay -1, and the cache drops what is
 * written there.
 * rows_off, row_pos and row_slot describe the new tokens as packed rows: the offsets
 * that the layer's calls take, each row's position, and its slot, page * page_size +
 * place in the page (-1: no page). Rows behind the last one are left alone.
 * copies: where a sequence's last page is not full and held by others too, it must not
 * be written: the sequence gets a page of its own and copies[b] = (old page, new page)
 * for c4s_kv_copy, else (-1, -1). Of sequences that hold a page together and all go on
 * (and nothing else holds it), the last one keeps it. Without copies nothing is looked
 * at: then no sequence may have such a page. (The page that is not to be had: the
 * sequence's entry becomes -1, its tokens there are lost, copies[b] is (-1, -1).) */
typedef struct c4s_grow {
  const int32_t* n_new;      /* [n_seqs], or NULL (1 each) */
  int32_t* rows_off;         /* [n_seqs + 1], or NULL */
  int32_t* row_pos;          /* [n_rows], or NULL; these two need rows_off, or n_new NULL */
  int32_t* row_slot;         /* [n_rows], or NULL */
  int32_t* copies;           /* [n_seqs][2], or NULL */
  int32_t n_rows;            /* room of row_pos and row_slot: rows from there on are not written */
} c4s_grow;

int c4s_pages_grow(c4s_ctx* ctx, const c4s_pages* pages, const c4s_grow* grow, void* stream);

/* lens[b] -= n_drop[b] (below 0: 0; at most to 0), and pages without a token are given back. */
int c4s_pages_trim(c4s_ctx* ctx, const c4s_pages* pages, const int32_t* n_drop, void* stream);

/* Sequences in groups of `width` (1 .. 32; n_seqs a multiple): sequence g * width + j
 * becomes what g * width + parent[g * width + j] was, length and pages (which they then
 * hold together); pages that nobody holds any more are given back. A parent outside
 * [0, width): the sequence is empty. */
int c4s_pages_fork(c4s_ctx* ctx, const c4s_pages* pages, const int32_t* parent, int32_t width, void* stream);

/* Page copies[i][0] of the cache into page copies[i][1], i < n; pairs with a number that
 * is no page are skipped. A page that is written must not be in another pair. */
int c4s_kv_copy(c4s_ctx* ctx, const c4s_kv_cache* cache, const int32_t* copies, int32_t n, void* stream);

/* ---- beams ----------------------------------------------------------------------------
 *
 * Rows in groups of `width`. With z the row's logits after repetition penalty and
 * temperature, as c4s_sample_rows applies them, every row r = g * width + j offers its
 * group for every token v the total
 *   score[r] + z[v] - log sum_u exp z[u]
 * (-inf where score or z is, and where it would be NaN, as for all of a row with NaN or +inf among its
 * z), a row that is done only its stop token, with its score as it is. The `width` largest totals of a group, equal ones by the lowest
 * (j, v), become its rows: parent j, token v, out_score the total, out_done whether the
 * parent was done or v is the stop token.
 * Totals are in 64 bits, of exponentials in 32: a row's log sum is off by up to
 *   2^-22 (1.5 + the mean of |z - the row's largest|, weighted by exp z),
 * 4e-7 to 2e-6, for all its tokens alike, and by a little else in a call of another number
 * of rows. Two rows' totals that lie nearer to each other may come in either order.
 * hist_bits and the states are carried along: row g * width + i of each output is row
 * g * width + out_parent[..] of its input, and out_hist_bits then has the token added,
 * unless the row was or is done. Outputs may be their inputs themselves.
 * A group begins with its first row's score 0 and the others' -inf. */
typedef struct c4s_beam_state {
  const void* src;           /* [rows][ld_src] 32-bit words, 4-byte aligned */
  void* dst;                 /* [rows][ld_dst], or src itself with its stride */
  int64_t ld_src, ld_dst;    /* >= words */
  int64_t words;             /* of a row, up to 2147483647; ceil(all states' and the history's words / 256) * n_groups up to 16777215 */
} c4s_beam_state;

enum { C4S_BEAM_STATES = 8 };

typedef struct c4s_beam {
  const void* logits;        /* [rows][ld] in dtype */
  int64_t ld;
  int32_t dtype;             /* C4S_DTYPE_F32 or C4S_DTYPE_BF16 */
  int32_t n_groups;          /* n_groups * width up to 1048576, n_groups up to 65536 */
  int32_t width;             /* 1 .. 32 */
  int32_t vocab;             /* 1 .. 1048576 */
  int32_t stop_token;        /* a token, or -1: none */
  int32_t n_states;          /* up to C4S_BEAM_STATES */
  const float* temperature;  /* [rows] or NULL */
  const float* rep_penalty;  /* [rows] or NULL; goes with hist_bits */
  const uint32_t* hist_bits; /* [rows][(vocab + 31) / 32] or NULL: the tokens that have come */
  uint32_t* out_hist_bits;   /* with hist_bits */
  const float* score;        /* [rows] */
  const uint8_t* done;       /* [rows] or NULL (none is); needs a stop token */
  float* out_score;          /* [rows] */
  uint8_t* out_done;         /* [rows] or NULL */
  int32_t* out_parent;       /* [rows] */
  int32_t* out_token;        /* [rows] */
  c4s_beam_state states[C4S_BEAM_STATES];
} c4s_beam;

int c4s_beam_step(c4s_ctx* ctx, const c4s_beam* beam, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* C4S_BATCH_H */
