// The paged key-value cache: rows written as bf16 or as 8-bit codes, and read
// back (include/c4s_layers.h has the layout).
//
// Both kernels take tiles of 16 packed rows of one head, 16 lanes a row (one
// DPP row of a wave, which is what the row's maximum is taken over). Keys keep
// their order: a lane's four dims go to the page as 8 bytes (bf16) or 4
// (codes), a row's lanes next to each other. Values lie in the page with their
// positions next to each other, so a tile of them passes through LDS, and a
// wave stores 4 dims of 16 positions at a time.

#include <hip/hip_runtime.h>

#include "c4s_layers.hpp"

namespace c4s {
namespace {

constexpr int kTile = 16;          // rows a workgroup takes
constexpr int kKvThreads = 256;
constexpr int kMaxDim = 256;

// Where packed row r lies in the cache: its page and place in it, or -1 when
// the row belongs to no sequence or its position has no page.
struct Place {
  int64_t page;
  int at;
};
__device__ __forceinline__ Place place_of(const KvArgs& c, const int32_t* lens, const int32_t* off, int n_rows, int r) {
  Place p{-1, 0};
  if (r >= n_rows) return p;
  int seq = r;
  int64_t pos;
  if (off) {
    int lo = 0, hi = c.n_seqs;   // the last sequence that starts at or before r
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (off[mid] <= r) lo = mid; else hi = mid;
    }
    seq = lo;
    const int end = off[seq + 1];
    if (r < off[seq] || r >= end) return p;
    pos = (int64_t)lens[seq] - (end - r);
  } else {
    if (seq >= c.n_seqs) return p;
    pos = (int64_t)lens[seq] - 1;
  }
  const int64_t i = pos >> c.page_shift;
  if (pos < 0 || i >= c.max_pages) return p;
  const int page = c.table[seq * c.table_ld + i];
  if (page < 0 || page >= c.n_pages) return p;
  p.page = page;
  p.at = (int)(pos & ((1 << c.page_shift) - 1));
  return p;
}

__device__ __forceinline__ float max16(float v) {   // over a row's 16 lanes
#pragma unroll
  for (int o = 8; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 16));
  return v;
}

__device__ __forceinline__ float from_bf16(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t to_bf16(float f) {   // round to nearest even
  return __builtin_bit_cast(uint16_t, (__bf16)f);
}

__global__ __launch_bounds__(kKvThreads) void k_kv_append(KvArgs c, KvRowsArgs rows) {
  __shared__ __align__(16) uint16_t tile[kMaxDim][kTile + 2];
  __shared__ Place places[kTile];
  const int head = blockIdx.y, row = threadIdx.x / 16, l = threadIdx.x % 16;
  const int r = blockIdx.x * kTile + row, dim = c.dim, ps = 1 << c.page_shift;
  if (threadIdx.x < kTile) places[threadIdx.x] = place_of(c, rows.lens, rows.off, rows.n_rows, blockIdx.x * kTile + threadIdx.x);
  __syncthreads();
  const Place p = places[row];
  const bool q8 = c.store == C4S_KV_Q8;
  const int64_t slot = (p.page * c.n_heads + head) * (int64_t)ps + p.at;   // (position, head) in the cache
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const uint16_t* src = static_cast<const uint16_t*>(which ? rows.v : rows.k) + (int64_t)r * (which ? rows.ldv : rows.ldk) + head * dim;
    uint2 raw[kMaxDim / 64];
    float top = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
      const int d = 64 * i + 4 * l;
      if (p.page < 0 || d >= dim) continue;
      raw[i] = *reinterpret_cast<const uint2*>(src + d);
      const float v[4] = {from_bf16(raw[i].x & 0xFFFFu), from_bf16(raw[i].x >> 16), from_bf16(raw[i].y & 0xFFFFu), from_bf16(raw[i].y >> 16)};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        top = fmaxf(top, fabsf(v[j]));
        finite = finite && v[j] - v[j] == 0.0f;
      }
    }
    float scale = 1.0f;
    if (q8) {
      // a value that is not finite makes the scale NaN, and so the row
      top = max16(finite ? top : __builtin_inff());
      scale = top < __builtin_inff() ? top / 127.0f : __builtin_nanf("");
      if (p.page >= 0 && l == 0) (which ? c.v_scale : c.k_scale)[slot] = scale;
    }
#pragma unroll
    for (int i = 0; i < kMaxDim / 64; ++i) {
      const int d = 64 * i + 4 * l;
      if (p.page < 0 || d >= dim) continue;
      uint32_t h[4] = {raw[i].x & 0xFFFFu, raw[i].x >> 16, raw[i].y & 0xFFFFu, raw[i].y >> 16};
      if (q8) {
#pragma unroll
        for (int j = 0; j < 4; ++j)   // round to even; |value / scale| is at most 127 to within a rounding
          h[j] = scale > 0.0f ? (uint32_t)(int)fminf(fmaxf(rintf(from_bf16(h[j]) / scale), -127.0f), 127.0f) & 0xFFu : 0u;
      }
      if (which == 0) {
        if (q8)
          *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(c.k) + slot * dim + d) = h[0] | h[1] << 8 | h[2] << 16 | h[3] << 24;
        else
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(c.k) + slot * dim + d) = raw[i];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) tile[d + j][row] = (uint16_t)h[j];
      }
    }
  }
  __syncthreads();
  const Place pv = places[threadIdx.x % 16];
  if (pv.page < 0) return;
  const int64_t base = (pv.page * c.n_heads + head) * (int64_t)ps * dim + pv.at;
  for (int d = threadIdx.x / 16; d < dim; d += kKvThreads / 16) {
    const uint16_t h = tile[d][threadIdx.x % 16];
    if (q8) static_cast<uint8_t*>(c.v)[base + (int64_t)d * ps] = (uint8_t)h;
    else static_cast<uint16_t*>(c.v)[base + (int64_t)d * ps] = h;
  }
}

__global__ __launch_bounds__(kKvThreads) void k_kv_read(KvArgs c, KvRowsArgs rows) {
  __shared__ __align__(16) float tile[kMaxDim][kTile + 1];
  __shared__ Place places[kTile];
  const int head = blockIdx.y, row = threadIdx.x / 16, l = threadIdx.x % 16;
  const int r = blockIdx.x * kTile + row, dim = c.dim, ps = 1 << c.page_shift;
  if (threadIdx.x < kTile) places[threadIdx.x] = place_of(c, rows.lens, rows.off, rows.n_rows, blockIdx.x * kTile + threadIdx.x);
  // a row between two sequences' rows, or behind the last, is not the call's to write
  __shared__ bool member[kTile];
  if (threadIdx.x < kTile) {
    const int rr = blockIdx.x * kTile + threadIdx.x;
    member[threadIdx.x] = rr < rows.n_rows && (!rows.off || (rr >= rows.off[0] && rr < rows.off[c.n_seqs]));
  }
  __syncthreads();
  const bool q8 = c.store == C4S_KV_Q8;
  {
    const Place pv = places[threadIdx.x % 16];
    const int64_t slot = (pv.page * c.n_heads + head) * (int64_t)ps + pv.at;
    const int64_t base = (pv.page * c.n_heads + head) * (int64_t)ps * dim + pv.at;
    const float scale = q8 && pv.page >= 0 ? c.v_scale[slot] : 1.0f;
    for (int d = threadIdx.x / 16; d < dim; d += kKvThreads / 16) {
      float v = 0.0f;
      if (pv.page >= 0)
        v = q8 ? (float)static_cast<const int8_t*>(c.v)[base + (int64_t)d * ps] * scale
               : from_bf16(static_cast<const uint16_t*>(c.v)[base + (int64_t)d * ps]);
      tile[d][threadIdx.x % 16] = v;
    }
  }
  __syncthreads();
  if (!member[row]) return;
  const Place p = places[row];
  const int64_t slot = (p.page * c.n_heads + head) * (int64_t)ps + p.at;
  const float scale = q8 && p.page >= 0 ? c.k_scale[slot] : 1.0f;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    for (int d = 4 * l; d < dim; d += 64) {
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (which) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = tile[d + j][row];
      } else if (p.page >= 0 && q8) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(c.k) + slot * dim + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)(int8_t)(w >> (8 * j)) * scale;
      } else if (p.page >= 0) {
        const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(c.k) + slot * dim + d);
        v[0] = from_bf16(w.x & 0xFFFFu);
        v[1] = from_bf16(w.x >> 16);
        v[2] = from_bf16(w.y & 0xFFFFu);
        v[3] = from_bf16(w.y >> 16);
      }
      void* out = which ? rows.v : rows.k;
      const int64_t o = (int64_t)r * (which ? rows.ldv : rows.ldk) + head * dim + d;
      if (rows.f32)
        *reinterpret_cast<float4*>(static_cast<float*>(out) + o) = make_float4(v[0], v[1], v[2], v[3]);
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + o) =
            make_uint2(to_bf16(v[0]) | to_bf16(v[1]) << 16, to_bf16(v[2]) | to_bf16(v[3]) << 16);
    }
  }
}

}  // namespace

hipError_t launch_kv_append(const KvArgs& c, const KvRowsArgs& r, hipStream_t s) {
  hipLaunchKernelGGL(k_kv_append, dim3((r.n_rows + kTile - 1) / kTile, c.n_heads), dim3(kKvThreads), 0, s, c, r);
  return hipGetLastError();
}

hipError_t launch_kv_read(const KvArgs& c, const KvRowsArgs& r, hipStream_t s) {
  hipLaunchKernelGGL(k_kv_read, dim3((r.n_rows + kTile - 1) / kTile, c.n_heads), dim3(kKvThreads), 0, s, c, r);
  return hipGetLastError();
}

}  // namespace c4s
