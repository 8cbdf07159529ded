// Launches of the batch's operators (include/c4s_batch.h), shared by their
// kernels and the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/c4s_batch.h"
#include "c4s_layers.hpp"

namespace c4s {

constexpr int kPagesSeqs = 4096;   // sequences of c4s_pages, whose numbers of pages lie in LDS
constexpr int kBeamWidth = 32;

hipError_t launch_rope(const c4s_rope_desc& a, hipStream_t s);
hipError_t launch_pages_grow(const c4s_pages& p, const c4s_grow& g, hipStream_t s);
hipError_t launch_pages_trim(const c4s_pages& p, const int32_t* n_drop, hipStream_t s);
hipError_t launch_pages_fork(const c4s_pages& p, const int32_t* parent, int width, hipStream_t s);
hipError_t launch_kv_copy(const KvArgs& c, const int32_t* copies, int n, hipStream_t s);
LayerSpace beam_space(const c4s_beam& a);
hipError_t launch_beam(const c4s_beam& a, uint32_t* counters, float* space, hipStream_t s);

}  // namespace c4s
