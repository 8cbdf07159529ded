// Launch descriptors of the decoder layer's operators, shared by their kernels
// and the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/c4s_layers.h"
#include "c4s_internal.h"

namespace c4s {

// What the kernels need of a cache.
struct KvArgs {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  const int32_t* table;
  int64_t table_ld;
  int n_seqs, max_pages, n_pages, page_shift, n_heads, dim, store;
};

struct KvRowsArgs {
  void* k;
  void* v;
  int64_t ldk, ldv;
  const int32_t* lens;
  const int32_t* off;
  int n_rows;
  bool f32;
};

struct AttnArgs {
  KvArgs c;
  const uint16_t* q;
  int64_t ldq;
  uint16_t* out;
  int64_t ld_out;
  float* lse;
  const int32_t* lens;
  const int32_t* off;
  const int32_t* first;
  int n_rows, max_new, n_heads, shared;   // shared: query heads a key head
  float scale;
};

// What a call needs of its stream's workspace: counters that are zero between
// calls (a kernel that uses them leaves them so), and floats.
struct LayerSpace {
  int64_t counters = 0, floats = 0;
};

hipError_t launch_block_norm(const c4s_norm& a, hipStream_t s);
LayerSpace linear_space(const c4s_linear_desc& a);
hipError_t launch_linear(const c4s_linear_desc& a, uint32_t* counters, float* space, hipStream_t s);
hipError_t launch_kv_append(const KvArgs& c, const KvRowsArgs& r, hipStream_t s);
hipError_t launch_kv_read(const KvArgs& c, const KvRowsArgs& r, hipStream_t s);
LayerSpace attn_space(const AttnArgs& a);
hipError_t launch_attn(const AttnArgs& a, uint32_t* counters, float* space, hipStream_t s);

}  // namespace c4s
