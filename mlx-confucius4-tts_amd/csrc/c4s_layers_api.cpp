// C ABI of the decoder layer's operators (declarations and contracts in
// include/c4s_layers.h). Host side only: argument checks, workspaces, dispatch.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>

#include "../../include/c4s_layers.h"
#include "c4s_ctx.hpp"
#include "c4s_layers.hpp"

using c4s::DeviceGuard;
using c4s::fail;
using c4s::hip_fail;

namespace {

bool is_dtype(int32_t d) { return d == C4S_DTYPE_F32 || d == C4S_DTYPE_BF16; }
uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

int launched(c4s_ctx* ctx, hipError_t e, const char* what) {
  return e == hipSuccess ? C4S_OK : hip_fail(ctx, e, what);
}

// Runs `body` with the context's device current; nothing is thrown through the ABI.
template <class Body>
int entry(c4s_ctx* ctx, const void* desc, const char* what, Body body) {
  if (!ctx) return C4S_EINVAL;
  try {
    if (!desc) return fail(ctx, C4S_EINVAL, std::string(what) + ": descriptor is NULL");
    return body();
  } catch (const std::bad_alloc&) {
    return C4S_ENOMEM;
  } catch (...) {
    return C4S_EHIP;
  }
}

// As queue(), with `need` of the stream's workspace: launch(counters, floats).
template <class Launch>
int queue_with(c4s_ctx* ctx, const c4s::LayerSpace& need, hipStream_t s, const char* what, Launch launch) {
  DeviceGuard g(ctx->device);
  if (g.err != hipSuccess) return hip_fail(ctx, g.err, "hipSetDevice");
  if (need.floats == 0) return launched(ctx, launch(nullptr, nullptr), what);
  if (need.counters * 4 > (int64_t)c4s::kLayerZeroed) return fail(ctx, C4S_EINVAL, std::string(what) + ": too many parts");
  ctx->layer_ws.runtime().stream = ctx->host_stream;
  void* ws = nullptr;
  const int rc = c4s::pool_take(ctx, ctx->layer_ws, s, c4s::kLayerZeroed + (size_t)need.floats * 4, "layer workspace", &ws);
  if (rc) return rc;
  const hipError_t e = launch(static_cast<uint32_t*>(ws), reinterpret_cast<float*>(static_cast<char*>(ws) + c4s::kLayerZeroed));
  ctx->layer_ws.queued(s, c4s::is_capturing(s));
  return launched(ctx, e, what);
}

template <class Launch>
int queue(c4s_ctx* ctx, const char* what, Launch launch) {
  DeviceGuard g(ctx->device);
  if (g.err != hipSuccess) return hip_fail(ctx, g.err, "hipSetDevice");
  return launched(ctx, launch(), what);
}

int check_norm(c4s_ctx* ctx, const c4s_norm* a) {
  if (a->M < 0 || a->D < 1 || a->D > 16384) return fail(ctx, C4S_EINVAL, "block_norm: needs M >= 0, D in 1 .. 16384");
  if (a->M == 0) return C4S_OK;
  if (a->kind != C4S_NORM_LAYER && a->kind != C4S_NORM_RMS) return fail(ctx, C4S_EINVAL, "block_norm: unknown kind");
  if (!a->x || (!a->x_out && !a->out)) return fail(ctx, C4S_EINVAL, "block_norm: x, or both outputs, NULL");
  if (!is_dtype(a->x_dtype) || !is_dtype(a->out_dtype) || (a->y && !is_dtype(a->y_dtype)))
    return fail(ctx, C4S_EINVAL, "block_norm: unknown dtype");
  if (!(a->eps >= 0.0f)) return fail(ctx, C4S_EINVAL, "block_norm: eps is negative or NaN");
  if (!a->y && (a->post || a->gate)) return fail(ctx, C4S_EINVAL, "block_norm: post or gate without y");
  if (a->gate && (a->gate_rows < 1 || a->ld_gate < a->D))
    return fail(ctx, C4S_EINVAL, "block_norm: gate needs gate_rows >= 1 and ld_gate >= D");
  if (a->ldx < a->D || (a->y && a->ldy < a->D) || (a->x_out && a->ld_x_out < a->D) || (a->out && a->ld_out < a->D))
    return fail(ctx, C4S_EINVAL, "block_norm: a row stride is below D");
  return C4S_OK;
}

int check_linear(c4s_ctx* ctx, const c4s_linear_desc* a) {
  if (a->M < 0 || a->N < 1 || a->K < 8 || a->K % 8) return fail(ctx, C4S_EINVAL, "linear: needs M >= 0, N >= 1, K a positive multiple of 8");
  if (a->N > 1 << 22 || a->K > 1 << 22) return fail(ctx, C4S_EINVAL, "linear: N or K above 4194304");
  // rows are counted in 32 bits, up to a tile past the last; a grid has up to 2^32 threads, 256 a tile
  if (a->M > 1 << 30) return fail(ctx, C4S_EINVAL, "linear: M above 1073741824");
  if (((int64_t)a->M + 127) / 128 * ((a->N + 127) / 128) > (1 << 24) - 8)
    return fail(ctx, C4S_EINVAL, "linear: more than 16777208 tiles of 128 x 128 outputs");
  if (a->M == 0) return C4S_OK;
  if (!a->x || !a->weight || !a->out) return fail(ctx, C4S_EINVAL, "linear: required pointer is NULL");
  if (a->act < C4S_ACT_NONE || a->act > C4S_ACT_RELU) return fail(ctx, C4S_EINVAL, "linear: unknown activation");
  if (a->wdtype != C4S_W_BF16 && a->wdtype != C4S_W_Q8) return fail(ctx, C4S_EINVAL, "linear: weights are bf16 or 8-bit codes");
  if (a->wdtype == C4S_W_Q8) {
    if (!a->wscale || !a->wbias) return fail(ctx, C4S_EINVAL, "linear: 8-bit weights need wscale and wbias");
    if ((a->group != 32 && a->group != 64 && a->group != 128) || a->K % a->group)
      return fail(ctx, C4S_EINVAL, "linear: group must be 32, 64 or 128 and divide K");
  }
  if (!is_dtype(a->out_dtype) || (a->residual && !is_dtype(a->res_dtype))) return fail(ctx, C4S_EINVAL, "linear: unknown dtype");
  if (a->ldx > 1 << 22) return fail(ctx, C4S_EINVAL, "linear: ldx above 4194304");
  if (a->ldx < a->K || a->ld_out < a->N || (a->residual && a->ld_res < a->N))
    return fail(ctx, C4S_EINVAL, "linear: a row stride is below its row");
  if ((bits(a->x) & 15u) || (a->ldx & 7) || (bits(a->weight) & (a->wdtype == C4S_W_Q8 ? 7u : 15u)))
    return fail(ctx, C4S_EINVAL, "linear: rows of x and weight must start on 16 bytes (8-bit weights: 8)");
  return C4S_OK;
}

int check_cache(c4s_ctx* ctx, const c4s_kv_cache* c) {
  if (c->n_seqs < 0 || c->n_seqs > 65535 || c->n_pages < 1 || c->max_pages < 0 || c->table_ld < c->max_pages)
    return fail(ctx, C4S_EINVAL, "kv_cache: n_seqs, n_pages, max_pages or table_ld out of range");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return fail(ctx, C4S_EINVAL, "kv_cache: page_size must be 16, 32, 64, 128 or 256");
  if (c->head_dim < 16 || c->head_dim > 256 || c->head_dim % 16)
    return fail(ctx, C4S_EINVAL, "kv_cache: head_dim must be a multiple of 16 up to 256");
  if (c->n_kv_heads < 1 || c->n_kv_heads > 65535) return fail(ctx, C4S_EINVAL, "kv_cache: n_kv_heads out of range");
  if ((int64_t)c->max_pages * c->page_size > 1 << 21) return fail(ctx, C4S_EINVAL, "kv_cache: more than 2097152 positions a sequence");
  if ((int64_t)c->n_kv_heads * c->page_size * c->head_dim > 1 << 29) return fail(ctx, C4S_EINVAL, "kv_cache: more than 536870912 values a page");
  if (!c->k || !c->v || (c->max_pages && !c->block_table)) return fail(ctx, C4S_EINVAL, "kv_cache: required pointer is NULL");
  if (c->store != C4S_KV_BF16 && c->store != C4S_KV_Q8) return fail(ctx, C4S_EINVAL, "kv_cache: unknown store");
  if (c->store == C4S_KV_Q8 && (!c->k_scale || !c->v_scale)) return fail(ctx, C4S_EINVAL, "kv_cache: 8-bit codes need k_scale and v_scale");
  uintptr_t al = bits(c->k) | bits(c->v);
  if (c->store == C4S_KV_Q8) al |= bits(c->k_scale) | bits(c->v_scale);
  if (al & 15u) return fail(ctx, C4S_EINVAL, "kv_cache: k, v and their scales must be 16-byte aligned");
  return C4S_OK;
}

c4s::KvArgs to_args(const c4s_kv_cache* c) {
  int shift = 0;
  while ((1 << shift) < c->page_size) ++shift;
  return c4s::KvArgs{c->k,       c->v,          c->k_scale,    c->v_scale,    c->block_table, c->table_ld, c->n_seqs,
                     c->max_pages, c->n_pages, shift, c->n_kv_heads, c->head_dim, c->store};
}

int check_rows(c4s_ctx* ctx, const c4s_kv_cache* c, const c4s_kv_rows* r, bool read) {
  int rc = check_cache(ctx, c);
  if (rc) return rc;
  if (r->n_rows < 0) return fail(ctx, C4S_EINVAL, "kv_rows: n_rows < 0");
  if (r->n_rows == 0) return C4S_OK;
  if (!r->k || !r->v || !r->lens) return fail(ctx, C4S_EINVAL, "kv_rows: required pointer is NULL");
  if (r->dtype != C4S_DTYPE_BF16 && !(read && r->dtype == C4S_DTYPE_F32))
    return fail(ctx, C4S_EINVAL, "kv_rows: rows are bf16 (read: or f32)");
  const int64_t w = (int64_t)c->n_kv_heads * c->head_dim;
  if (r->ldk < w || r->ldv < w) return fail(ctx, C4S_EINVAL, "kv_rows: a row stride is below n_kv_heads * head_dim");
  const uintptr_t mask = r->dtype == C4S_DTYPE_F32 ? 15u : 7u;
  if (((bits(r->k) | bits(r->v)) & mask) || ((r->ldk | r->ldv) & 3))
    return fail(ctx, C4S_EINVAL, "kv_rows: rows must start on 8 bytes (f32: 16)");
  if ((int64_t)r->n_rows * c->n_kv_heads > 1 << 29) return fail(ctx, C4S_EINVAL, "kv_rows: n_rows * n_kv_heads above 536870912");
  if (!r->rows_off && r->n_rows > c->n_seqs) return fail(ctx, C4S_EINVAL, "kv_rows: more rows than sequences without rows_off");
  return C4S_OK;
}

c4s::KvRowsArgs to_args(const c4s_kv_rows* r) {
  return c4s::KvRowsArgs{r->k, r->v, r->ldk, r->ldv, r->lens, r->rows_off, r->n_rows, r->dtype == C4S_DTYPE_F32};
}

// Rows a sequence has at most: one without rows_off, whatever max_new says, and never more than there are.
int32_t new_rows(const c4s_attn_desc* a) { return a->rows_off ? std::min(a->max_new, a->n_rows) : 1; }

int check_attn(c4s_ctx* ctx, const c4s_kv_cache* c, const c4s_attn_desc* a) {
  int rc = check_cache(ctx, c);
  if (rc) return rc;
  if (a->n_rows < 0 || (a->rows_off && a->max_new < 0)) return fail(ctx, C4S_EINVAL, "attn: n_rows or max_new < 0");
  if (a->n_heads < 1 || a->n_heads % c->n_kv_heads) return fail(ctx, C4S_EINVAL, "attn: n_heads must be a multiple of n_kv_heads");
  if (a->n_rows == 0) return C4S_OK;
  if (!a->q || !a->out || !a->lens) return fail(ctx, C4S_EINVAL, "attn: required pointer is NULL");
  const int64_t w = (int64_t)a->n_heads * c->head_dim;
  if (a->ldq < w || a->ld_out < w) return fail(ctx, C4S_EINVAL, "attn: a row stride is below n_heads * head_dim");
  if ((bits(a->q) & 15u) || (a->ldq & 7) || (bits(a->out) & 7u) || (a->ld_out & 3))
    return fail(ctx, C4S_EINVAL, "attn: rows of q must start on 16 bytes, rows of out on 8");
  if (!a->rows_off && a->n_rows > c->n_seqs) return fail(ctx, C4S_EINVAL, "attn: more rows than sequences without rows_off");
  if (!(a->scale - a->scale == 0.0f)) return fail(ctx, C4S_EINVAL, "attn: scale is not finite");
  if ((int64_t)new_rows(a) * a->n_heads > 1 << 29) return fail(ctx, C4S_EINVAL, "attn: max_new * n_heads above 536870912");
  return C4S_OK;
}

}  // namespace

extern "C" {

int c4s_block_norm(c4s_ctx* ctx, const c4s_norm* norm, void* stream) {
  return entry(ctx, norm, "block_norm", [&] {
    const int rc = check_norm(ctx, norm);
    if (rc || norm->M == 0) return rc;
    return queue(ctx, "block_norm launch", [&] { return c4s::launch_block_norm(*norm, static_cast<hipStream_t>(stream)); });
  });
}

int c4s_linear(c4s_ctx* ctx, const c4s_linear_desc* lin, void* stream) {
  return entry(ctx, lin, "linear", [&] {
    const int rc = check_linear(ctx, lin);
    if (rc || lin->M == 0) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return queue_with(ctx, c4s::linear_space(*lin), s, "linear launch",
                      [&](uint32_t* n, float* f) { return c4s::launch_linear(*lin, n, f, s); });
  });
}

int c4s_kv_append(c4s_ctx* ctx, const c4s_kv_cache* cache, const c4s_kv_rows* rows, void* stream) {
  return entry(ctx, cache && rows ? cache : nullptr, "kv_append", [&] {
    const int rc = check_rows(ctx, cache, rows, false);
    if (rc || rows->n_rows == 0 || cache->n_seqs == 0) return rc;
    return queue(ctx, "kv_append launch", [&] {
      return c4s::launch_kv_append(to_args(cache), to_args(rows), static_cast<hipStream_t>(stream));
    });
  });
}

int c4s_kv_read(c4s_ctx* ctx, const c4s_kv_cache* cache, const c4s_kv_rows* rows, void* stream) {
  return entry(ctx, cache && rows ? cache : nullptr, "kv_read", [&] {
    const int rc = check_rows(ctx, cache, rows, true);
    if (rc || rows->n_rows == 0 || cache->n_seqs == 0) return rc;
    return queue(ctx, "kv_read launch", [&] {
      return c4s::launch_kv_read(to_args(cache), to_args(rows), static_cast<hipStream_t>(stream));
    });
  });
}

int c4s_attn(c4s_ctx* ctx, const c4s_kv_cache* cache, const c4s_attn_desc* attn, void* stream) {
  return entry(ctx, cache && attn ? cache : nullptr, "attn", [&] {
    const int rc = check_attn(ctx, cache, attn);
    if (rc || attn->n_rows == 0 || new_rows(attn) == 0 || cache->n_seqs == 0) return rc;
    c4s::AttnArgs a{};
    a.c = to_args(cache);
    a.q = attn->q;
    a.ldq = attn->ldq;
    a.out = attn->out;
    a.ld_out = attn->ld_out;
    a.lse = attn->lse;
    a.lens = attn->lens;
    a.off = attn->rows_off;
    a.first = attn->first;
    a.n_rows = attn->n_rows;
    a.max_new = new_rows(attn);
    a.n_heads = attn->n_heads;
    a.shared = attn->n_heads / cache->n_kv_heads;
    a.scale = attn->scale;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return queue_with(ctx, c4s::attn_space(a), s, "attn launch",
                      [&](uint32_t* n, float* f) { return c4s::launch_attn(a, n, f, s); });
  });
}

}  // extern "C"
