// What the C-ABI entry points of the decoder's operators share: descriptor and
// exception guards, workspaces, checks of a cache. Host side only.
#pragma once

#include <hip/hip_runtime.h>

#include <new>

#include "../../include/c4s_layers.h"
#include "c4s_ctx.hpp"
#include "c4s_layers.hpp"

namespace c4s {

inline bool is_dtype(int32_t d) { return d == C4S_DTYPE_F32 || d == C4S_DTYPE_BF16; }
inline uintptr_t bits(const void* p) { return reinterpret_cast<uintptr_t>(p); }

inline int launched(c4s_ctx* ctx, hipError_t e, const char* what) {
  return e == hipSuccess ? C4S_OK : hip_fail(ctx, e, what);
}

// Runs `body`; nothing is thrown through the ABI.
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
int queue_with(c4s_ctx* ctx, const LayerSpace& need, hipStream_t s, const char* what, Launch launch) {
  DeviceGuard g(ctx->device);
  if (g.err != hipSuccess) return hip_fail(ctx, g.err, "hipSetDevice");
  if (need.floats == 0) return launched(ctx, launch(nullptr, nullptr), what);
  if (need.counters * 4 > (int64_t)kLayerZeroed) return fail(ctx, C4S_EINVAL, std::string(what) + ": too many parts");
  ctx->layer_ws.runtime().stream = ctx->host_stream;
  void* ws = nullptr;
  const int rc = pool_take(ctx, ctx->layer_ws, s, kLayerZeroed + (size_t)need.floats * 4, "layer workspace", &ws);
  if (rc) return rc;
  const hipError_t e = launch(static_cast<uint32_t*>(ws), reinterpret_cast<float*>(static_cast<char*>(ws) + kLayerZeroed));
  ctx->layer_ws.queued(s, is_capturing(s));
  return launched(ctx, e, what);
}

template <class Launch>
int queue(c4s_ctx* ctx, const char* what, Launch launch) {
  DeviceGuard g(ctx->device);
  if (g.err != hipSuccess) return hip_fail(ctx, g.err, "hipSetDevice");
  return launched(ctx, launch(), what);
}

inline int check_cache(c4s_ctx* ctx, const c4s_kv_cache* c) {
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
  if (c->store != C4S_KV_BF16 && c->store != C4S_KV_Q8 && c->store != C4S_KV_Q4) return fail(ctx, C4S_EINVAL, "kv_cache: unknown store");
  if (c->store == C4S_KV_Q4 && c->head_dim % 32) return fail(ctx, C4S_EINVAL, "kv_cache: 4-bit codes need a head_dim that is a multiple of 32");
  if (c->store != C4S_KV_BF16 && (!c->k_scale || !c->v_scale)) return fail(ctx, C4S_EINVAL, "kv_cache: 8-bit and 4-bit codes need k_scale and v_scale");
  uintptr_t al = bits(c->k) | bits(c->v);
  if (c->store != C4S_KV_BF16) al |= bits(c->k_scale) | bits(c->v_scale);
  if (al & 15u) return fail(ctx, C4S_EINVAL, "kv_cache: k, v and their scales must be 16-byte aligned");
  return C4S_OK;
}

inline KvArgs to_args(const c4s_kv_cache* c) {
  int shift = 0;
  while ((1 << shift) < c->page_size) ++shift;
  return KvArgs{c->k,       c->v,          c->k_scale,    c->v_scale,    c->block_table, c->table_ld, c->n_seqs,
                c->max_pages, c->n_pages, shift, c->n_kv_heads, c->head_dim, c->store};
}

}  // namespace c4s
