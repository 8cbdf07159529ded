// Norms around a block, with the residual stream between them (block_norm,
// include/c4s_layers.h): r = x + s g (.) u, u = y or norm(y); x_out = r; out =
// norm(r).
//
// A row stays in registers from the load to the last store, so x, y and the
// outputs pass through memory once (at least 8 bytes an element with bf16
// throughout: HBM-bound for many rows, one load's and two reductions' latency
// for few). The variance is taken over v - mean in a second sum over the
// registers, so a mean that is large against the deviations costs no digits.
// All sums are fp32, and out is the norm of r before x_out's rounding: that
// rounding then reaches the next block once, through the stream, and not twice.
//
// Stores pass the caches by: 16400 rows take 51 us with stores that stay in them,
// since a large call's outputs push its inputs out before they are read.
//
// Four elements are loaded and stored at a time, wherever rows begin (the
// hardware takes such accesses at any address that suits one element); a row
// whose length is not a multiple of four ends with single ones.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "c4s_layers.hpp"

namespace c4s {
namespace {

typedef float Float4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Half4 __attribute__((ext_vector_type(2), aligned(2)));   // four bf16

__device__ __forceinline__ float from_bf16(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

__device__ __forceinline__ void values(Half4 w, float (&v)[4]) {
  v[0] = from_bf16(w[0] & 0xFFFFu);
  v[1] = __uint_as_float(w[0] & 0xFFFF0000u);
  v[2] = from_bf16(w[1] & 0xFFFFu);
  v[3] = __uint_as_float(w[1] & 0xFFFF0000u);
}
__device__ __forceinline__ void values(Float4 w, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = w[j];
}

// Elements i .. i + 3 of p, in bf16 or fp32; those from n on are 0.
template <bool BF>
__device__ __forceinline__ void load(const void* p, int64_t i, int n, float (&v)[4]) {
  const uint16_t* h = static_cast<const uint16_t*>(p) + i;
  const float* f = static_cast<const float*>(p) + i;
  if (n >= 4) {
    if constexpr (BF) values(*reinterpret_cast<const Half4*>(h), v);
    else values(*reinterpret_cast<const Float4*>(f), v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? (BF ? from_bf16(h[j]) : f[j]) : 0.0f;
  }
}
__device__ __forceinline__ void store(void* p, bool bf, int64_t i, int n, const float (&v)[4]) {
  uint16_t* h = static_cast<uint16_t*>(p) + i;
  float* f = static_cast<float*>(p) + i;
  if (n >= 4) {
    if (bf)
      __builtin_nontemporal_store(Half4{to_bf16(v[0]) | to_bf16(v[1]) << 16, to_bf16(v[2]) | to_bf16(v[3]) << 16}, reinterpret_cast<Half4*>(h));
    else
      __builtin_nontemporal_store(Float4{v[0], v[1], v[2], v[3]}, reinterpret_cast<Float4*>(f));
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < n) {
        if (bf) h[j] = (uint16_t)to_bf16(v[j]);
        else f[j] = v[j];
      }
  }
}

// Sum over a wave, in all its lanes: neighbours, quads, halves of a row of 16
// lanes and rows by DPP, then the rows by exchange.
template <int CTRL>
__device__ __forceinline__ float plus_dpp(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = plus_dpp<0xB1>(v);    // quad_perm 1 0 3 2
  v = plus_dpp<0x4E>(v);    // quad_perm 2 3 0 1
  v = plus_dpp<0x141>(v);   // row_half_mirror
  v = plus_dpp<0x140>(v);   // row_mirror
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Sum over the T threads of a row; the same value in all of them. `part`: T / 64
// floats, another one's for each sum of a row (one barrier a sum).
template <int T>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = wave_sum(v);
  if constexpr (T > 64) {
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += part[w];
  }
  return v;
}

// T threads a row, each of them E pieces of four elements. TAIL: D is not a multiple of four.
template <int T, int E, bool TAIL>
struct Row {
  float v[E][4];
  int D, t;
  // f(e, i, n): piece e, elements i .. i + n - 1.
  template <class F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = (e * T + t) * 4;
      if (i < D) f(e, i, TAIL ? D - i : 4);
    }
  }
  // v becomes (v - mean) / sqrt(var + eps), or v / sqrt(mean of squares + eps); part: two sums' floats.
  __device__ __forceinline__ void norm(int kind, float eps, float* part) {
    if (kind == C4S_NORM_LAYER) {
      float s = 0.0f;
      each([&](int e, int, int) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s += v[e][j];
      });
      const float mean = row_sum<T>(s, part) / (float)D;
      each([&](int e, int, int n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[e][j] = !TAIL || j < n ? v[e][j] - mean : 0.0f;
      });
    }
    float q = 0.0f;
    each([&](int e, int, int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) q = __builtin_fmaf(v[e][j], v[e][j], q);
    });
    const float inv = 1.0f / sqrtf(row_sum<T>(q, part + T / 64) / (float)D + eps);
    each([&](int e, int, int) {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[e][j] *= inv;
    });
  }
  // v becomes v gamma + beta (absent: 1, 0).
  __device__ __forceinline__ void scaled(const float* gamma, const float* beta) {
    each([&](int e, int i, int n) {
      float g[4] = {1.0f, 1.0f, 1.0f, 1.0f}, b[4] = {};
      if (gamma) load<false>(gamma, i, n, g);
      if (beta) load<false>(beta, i, n, b);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[e][j] = __builtin_fmaf(v[e][j], g[j], b[j]);
    });
  }
};

constexpr int kNormThreads = 256;

// A row a wave (T = 64) or a workgroup. X, Y: whether x and y are bf16.
template <int T, int E, bool TAIL, bool X, bool Y>
__global__ __launch_bounds__(T > kNormThreads ? T : kNormThreads) void k_block_norm(c4s_norm a) {
  constexpr int kRows = T < kNormThreads ? kNormThreads / T : 1;
  __shared__ float part[4 * (T / 64)];
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kRows + (kRows > 1 ? (int)threadIdx.x / T : 0);
  if (row >= a.M) return;   // whole waves: with T > 64 a workgroup is one row
  const int m = (int)row;
  Row<T, E, TAIL> r;
  r.D = a.D;
  r.t = threadIdx.x % T;
  const int64_t x0 = (int64_t)m * a.ldx;
  if (a.y) {
    const int64_t y0 = (int64_t)m * a.ldy, g0 = a.gate ? (int64_t)(m / a.gate_rows) * a.ld_gate : 0;
    float x[E][4];
    r.each([&](int e, int i, int n) { load<X>(a.x, x0 + i, n, x[e]); });
    r.each([&](int e, int i, int n) { load<Y>(a.y, y0 + i, n, r.v[e]); });
    if (a.post) {
      r.norm(a.kind, a.eps, part);
      r.scaled(a.post_gamma, a.post_beta);
    }
    r.each([&](int e, int i, int n) {
      float g[4] = {1.0f, 1.0f, 1.0f, 1.0f};
      if (a.gate) load<false>(a.gate, g0 + i, n, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.v[e][j] = __builtin_fmaf(a.res_scale * g[j], r.v[e][j], x[e][j]);
    });
  } else {
    r.each([&](int e, int i, int n) { load<X>(a.x, x0 + i, n, r.v[e]); });
  }
  if (a.x_out) r.each([&](int e, int i, int n) { store(a.x_out, X, (int64_t)m * a.ld_x_out + i, n, r.v[e]); });
  if (!a.out) return;
  if constexpr (TAIL)   // a norm's and a gate's padding may have left something
    r.each([&](int e, int, int n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) r.v[e][j] = j < n ? r.v[e][j] : 0.0f;
    });
  r.norm(a.kind, a.eps, part + 2 * (T / 64));
  r.scaled(a.gamma, a.beta);
  r.each([&](int e, int i, int n) { store(a.out, a.out_dtype == C4S_DTYPE_BF16, (int64_t)m * a.ld_out + i, n, r.v[e]); });
}

template <int T, int E, bool TAIL>
hipError_t launch(const c4s_norm& a, hipStream_t s) {
  constexpr int kRows = T < kNormThreads ? kNormThreads / T : 1;
  const bool x = a.x_dtype == C4S_DTYPE_BF16, y = a.y && a.y_dtype == C4S_DTYPE_BF16;
  // a grid has up to 2^32 threads in a dimension
  const uint32_t groups = ((uint32_t)a.M + kRows - 1) / kRows, wide = std::min(groups, 1u << 20);
  const dim3 grid(wide, (groups + wide - 1) / wide), block(std::max(T, kNormThreads));
  if (x && y) hipLaunchKernelGGL((k_block_norm<T, E, TAIL, true, true>), grid, block, 0, s, a);
  else if (x) hipLaunchKernelGGL((k_block_norm<T, E, TAIL, true, false>), grid, block, 0, s, a);
  else if (y) hipLaunchKernelGGL((k_block_norm<T, E, TAIL, false, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((k_block_norm<T, E, TAIL, false, false>), grid, block, 0, s, a);
  return hipGetLastError();
}
template <int T, int E>
hipError_t launch(const c4s_norm& a, hipStream_t s) {
  return a.D % 4 ? launch<T, E, true>(a, s) : launch<T, E, false>(a, s);
}

__global__ void k_zero(uint32_t* p, size_t n) {
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0u;
}

}  // namespace

hipError_t launch_zero(void* p, size_t bytes, hipStream_t s) {
  hipLaunchKernelGGL(k_zero, dim3(64), dim3(256), 0, s, static_cast<uint32_t*>(p), bytes / 4);
  return hipGetLastError();
}

// A workgroup a row for few rows, where the row's own latency counts (1 row of
// 1280: 2.9 us, a wave a row 4.3; 1000 rows 4.5 and 6.1), and for long ones; a
// wave a row for many (16400 rows of 1280, bf16, a norm on both sides, gates: 36
// us, 4.7 TB/s, and 41; a copy reaches 5.4).
hipError_t launch_block_norm(const c4s_norm& a, hipStream_t s) {
  if (a.M <= 2048 && a.D > 256) {
    if (a.D <= 2048) return launch<256, 2>(a, s);
    if (a.D <= 8192) return launch<1024, 2>(a, s);
    return launch<1024, 4>(a, s);
  }
  if (a.D <= 512) return launch<64, 2>(a, s);
  if (a.D <= 1280) return launch<64, 5>(a, s);
  if (a.D <= 2048) return launch<64, 8>(a, s);
  if (a.D <= 8192) return launch<256, 8>(a, s);
  return launch<1024, 4>(a, s);
}

}  // namespace c4s
