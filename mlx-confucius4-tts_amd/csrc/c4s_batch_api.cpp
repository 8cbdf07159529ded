// C ABI of the batch's operators (declarations and contracts in
// include/c4s_batch.h). Host side only: argument checks, workspaces, dispatch.

#include <hip/hip_runtime.h>

#include "c4s_batch.hpp"
#include "c4s_entry.hpp"

using c4s::bits;
using c4s::check_cache;
using c4s::entry;
using c4s::fail;
using c4s::is_dtype;
using c4s::queue;
using c4s::queue_with;
using c4s::to_args;

namespace {

int check_rope(c4s_ctx* ctx, const c4s_rope_desc* a) {
  if (a->n_rows < 0 || a->n_rows > 16777215) return fail(ctx, C4S_EINVAL, "rope: n_rows must be 0 .. 16777215");
  if (a->head_dim < 2 || a->head_dim > 1024 || a->rot_dim < 2 || a->rot_dim > a->head_dim || a->rot_dim % 2)
    return fail(ctx, C4S_EINVAL, "rope: needs head_dim up to 1024 and an even rot_dim in 2 .. head_dim");
  if (a->layout != C4S_ROPE_HALF && a->layout != C4S_ROPE_PAIRS) return fail(ctx, C4S_EINVAL, "rope: unknown layout");
  if (!is_dtype(a->dtype)) return fail(ctx, C4S_EINVAL, "rope: unknown dtype");
  if (!(a->scale - a->scale == 0.0f)) return fail(ctx, C4S_EINVAL, "rope: scale is not finite");
  if (a->n_rows == 0) return C4S_OK;
  if ((!a->q && !a->k) || !a->freq || (!a->pos && !a->lens && a->n_seqs)) return fail(ctx, C4S_EINVAL, "rope: required pointer is NULL");
  if ((a->q && !a->q_out) || (a->k && !a->k_out)) return fail(ctx, C4S_EINVAL, "rope: a tensor without its output");
  if ((a->q && (a->n_heads < 1 || a->n_heads > 65535)) || (a->k && (a->n_kv_heads < 1 || a->n_kv_heads > 65535)))
    return fail(ctx, C4S_EINVAL, "rope: heads out of range");
  const int64_t wq = (int64_t)a->n_heads * a->head_dim, wk = (int64_t)a->n_kv_heads * a->head_dim;
  if ((a->q && (a->ldq < wq || a->ldq_out < wq)) || (a->k && (a->ldk < wk || a->ldk_out < wk)))
    return fail(ctx, C4S_EINVAL, "rope: a row stride is below heads * head_dim");
  if ((a->q && a->q == a->q_out && a->ldq != a->ldq_out) || (a->k && a->k == a->k_out && a->ldk != a->ldk_out))
    return fail(ctx, C4S_EINVAL, "rope: in place, both strides are the same");
  const uintptr_t size = a->dtype == C4S_DTYPE_F32 ? 4 : 2;
  if ((bits(a->q) | bits(a->q_out) | bits(a->k) | bits(a->k_out)) & (size - 1))
    return fail(ctx, C4S_EINVAL, "rope: a tensor is not aligned to its type");
  if (bits(a->freq) & 7u) return fail(ctx, C4S_EINVAL, "rope: freq must be 8-byte aligned");
  if (!a->pos) {
    if (a->n_seqs < 0 || a->n_seqs > 65535) return fail(ctx, C4S_EINVAL, "rope: n_seqs out of range");
    if (!a->rows_off && a->n_seqs && a->n_rows > a->n_seqs) return fail(ctx, C4S_EINVAL, "rope: more rows than sequences without rows_off");
  }
  return C4S_OK;
}

int check_pages(c4s_ctx* ctx, const c4s_pages* p) {
  if (p->n_seqs < 0 || p->n_seqs > c4s::kPagesSeqs) return fail(ctx, C4S_EINVAL, "pages: n_seqs must be 0 .. 4096");
  if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1)))
    return fail(ctx, C4S_EINVAL, "pages: page_size must be 16, 32, 64, 128 or 256");
  if (p->n_pages < 1 || (int64_t)p->n_pages * p->page_size > INT32_MAX)
    return fail(ctx, C4S_EINVAL, "pages: n_pages out of range");
  if (p->max_pages < 0 || p->table_ld < p->max_pages || (int64_t)p->max_pages * p->page_size > 1 << 21)
    return fail(ctx, C4S_EINVAL, "pages: max_pages or table_ld out of range");
  if (p->n_seqs == 0) return C4S_OK;
  if ((p->max_pages && !p->block_table) || !p->lens || !p->refs || !p->free_bits)
    return fail(ctx, C4S_EINVAL, "pages: required pointer is NULL");
  if (bits(p->free_bits) & 15u) return fail(ctx, C4S_EINVAL, "pages: free_bits must be 16-byte aligned");
  return C4S_OK;
}

int check_grow(c4s_ctx* ctx, const c4s_pages* p, const c4s_grow* g) {
  const int rc = check_pages(ctx, p);
  if (rc) return rc;
  if (g->n_rows < 0) return fail(ctx, C4S_EINVAL, "pages_grow: n_rows < 0");
  if ((g->row_pos || g->row_slot) && g->n_new && !g->rows_off)
    return fail(ctx, C4S_EINVAL, "pages_grow: row_pos and row_slot with n_new need rows_off");
  if (bits(g->copies) & 7u) return fail(ctx, C4S_EINVAL, "pages_grow: copies must be 8-byte aligned");
  return C4S_OK;
}

int check_beam(c4s_ctx* ctx, const c4s_beam* a) {
  if (a->n_groups < 0 || a->n_groups > 65536) return fail(ctx, C4S_EINVAL, "beam_step: n_groups must be 0 .. 65536");
  if (a->width < 1 || a->width > c4s::kBeamWidth) return fail(ctx, C4S_EINVAL, "beam_step: width must be 1 .. 32");
  if ((int64_t)a->n_groups * a->width > 1 << 20) return fail(ctx, C4S_EINVAL, "beam_step: more than 1048576 rows");
  if (a->vocab < 1 || a->vocab > 1 << 20 || a->ld < a->vocab)
    return fail(ctx, C4S_EINVAL, "beam_step: needs vocab in 1 .. 1048576 and ld >= vocab");
  if (!is_dtype(a->dtype)) return fail(ctx, C4S_EINVAL, "beam_step: unknown dtype");
  if (a->stop_token < -1 || a->stop_token >= a->vocab) return fail(ctx, C4S_EINVAL, "beam_step: stop_token must be -1 or a token");
  if (a->done && a->stop_token < 0) return fail(ctx, C4S_EINVAL, "beam_step: done needs a stop token");
  if (a->n_states < 0 || a->n_states > C4S_BEAM_STATES) return fail(ctx, C4S_EINVAL, "beam_step: n_states must be 0 .. 8");
  if (a->n_groups == 0) return C4S_OK;
  if (!a->logits || !a->score || !a->out_score || !a->out_parent || !a->out_token)
    return fail(ctx, C4S_EINVAL, "beam_step: required pointer is NULL");
  if (bits(a->logits) & (a->dtype == C4S_DTYPE_F32 ? 3u : 1u)) return fail(ctx, C4S_EINVAL, "beam_step: logits are not aligned to their type");
  if (!a->hist_bits != !a->out_hist_bits || (a->rep_penalty && !a->hist_bits))
    return fail(ctx, C4S_EINVAL, "beam_step: rep_penalty needs hist_bits, and hist_bits and out_hist_bits go together");
  int64_t words = a->hist_bits ? (a->vocab + 31) / 32 : 0;
  for (int i = 0; i < a->n_states; ++i) {
    const c4s_beam_state& s = a->states[i];
    if (s.words < 0 || s.ld_src < s.words || s.ld_dst < s.words)
      return fail(ctx, C4S_EINVAL, "beam_step: a state's row stride is below its words");
    if (s.words && (!s.src || !s.dst || ((bits(s.src) | bits(s.dst)) & 3u)))
      return fail(ctx, C4S_EINVAL, "beam_step: a state is NULL or not 4-byte aligned");
    if (s.words && s.src == s.dst && s.ld_src != s.ld_dst)
      return fail(ctx, C4S_EINVAL, "beam_step: a state in place has one stride");
    if (s.words > INT32_MAX) return fail(ctx, C4S_EINVAL, "beam_step: a state has more than 2147483647 words a row");
    words += s.words;
  }
  if ((words + 255) / 256 * a->n_groups > (1 << 24) - 1)   // a grid has up to 2^32 threads
    return fail(ctx, C4S_EINVAL, "beam_step: more than 16777215 times 256 words of states, each group's rounded up");
  return C4S_OK;
}

}  // namespace

extern "C" {

int c4s_rope(c4s_ctx* ctx, const c4s_rope_desc* rope, void* stream) {
  return entry(ctx, rope, "rope", [&] {
    const int rc = check_rope(ctx, rope);
    if (rc || rope->n_rows == 0 || (!rope->pos && rope->n_seqs == 0)) return rc;
    return queue(ctx, "rope launch", [&] { return c4s::launch_rope(*rope, static_cast<hipStream_t>(stream)); });
  });
}

int c4s_pages_grow(c4s_ctx* ctx, const c4s_pages* pages, const c4s_grow* grow, void* stream) {
  return entry(ctx, pages && grow ? pages : nullptr, "pages_grow", [&] {
    const int rc = check_grow(ctx, pages, grow);
    if (rc || pages->n_seqs == 0) return rc;
    return queue(ctx, "pages_grow launch", [&] { return c4s::launch_pages_grow(*pages, *grow, static_cast<hipStream_t>(stream)); });
  });
}

int c4s_pages_trim(c4s_ctx* ctx, const c4s_pages* pages, const int32_t* n_drop, void* stream) {
  return entry(ctx, pages, "pages_trim", [&] {
    const int rc = check_pages(ctx, pages);
    if (rc || pages->n_seqs == 0) return rc;
    if (!n_drop) return fail(ctx, C4S_EINVAL, "pages_trim: n_drop is NULL");
    return queue(ctx, "pages_trim launch", [&] { return c4s::launch_pages_trim(*pages, n_drop, static_cast<hipStream_t>(stream)); });
  });
}

int c4s_pages_fork(c4s_ctx* ctx, const c4s_pages* pages, const int32_t* parent, int32_t width, void* stream) {
  return entry(ctx, pages, "pages_fork", [&] {
    const int rc = check_pages(ctx, pages);
    if (rc) return rc;
    if (width < 1 || width > c4s::kBeamWidth || pages->n_seqs % width)
      return fail(ctx, C4S_EINVAL, "pages_fork: width must be 1 .. 32 and divide n_seqs");
    if (pages->n_seqs == 0) return rc;
    if (!parent) return fail(ctx, C4S_EINVAL, "pages_fork: parent is NULL");
    return queue(ctx, "pages_fork launch", [&] { return c4s::launch_pages_fork(*pages, parent, width, static_cast<hipStream_t>(stream)); });
  });
}

int c4s_kv_copy(c4s_ctx* ctx, const c4s_kv_cache* cache, const int32_t* copies, int32_t n, void* stream) {
  return entry(ctx, cache, "kv_copy", [&] {
    const int rc = check_cache(ctx, cache);
    if (rc) return rc;
    if (n < 0 || n > 65535) return fail(ctx, C4S_EINVAL, "kv_copy: n must be 0 .. 65535");
    if (n == 0) return rc;
    if (!copies || (bits(copies) & 7u)) return fail(ctx, C4S_EINVAL, "kv_copy: copies is NULL or not 8-byte aligned");
    return queue(ctx, "kv_copy launch", [&] { return c4s::launch_kv_copy(to_args(cache), copies, n, static_cast<hipStream_t>(stream)); });
  });
}

int c4s_beam_step(c4s_ctx* ctx, const c4s_beam* beam, void* stream) {
  return entry(ctx, beam, "beam_step", [&] {
    const int rc = check_beam(ctx, beam);
    if (rc || beam->n_groups == 0) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return queue_with(ctx, c4s::beam_space(*beam), s, "beam_step launch",
                      [&](uint32_t* n, float* f) { return c4s::launch_beam(*beam, n, f, s); });
  });
}

}  // extern "C"
