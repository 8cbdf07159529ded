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

#include <hip/hip_runtime.h>

#include "c4s_layers.hpp"

namespace c4s {
namespace {

__device__ __forceinline__ float from_bf16(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

// V consecutive elements at p[i], in bf16 or fp32; V is 4 (8- or 16-byte accesses) or 1.
template <int V>
__device__ __forceinline__ void load(const void* p, bool bf16, int64_t i, float (&v)[V]) {
  if constexpr (V == 4) {
    if (bf16) {
      const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + i);
      v[0] = from_bf16(w.x & 0xFFFFu);
      v[1] = __uint_as_float(w.x & 0xFFFF0000u);
      v[2] = from_bf16(w.y & 0xFFFFu);
      v[3] = __uint_as_float(w.y & 0xFFFF0000u);
    } else {
      const float4 w = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
      v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
    }
  } else {
    v[0] = bf16 ? from_bf16(static_cast<const uint16_t*>(p)[i]) : static_cast<const float*>(p)[i];
  }
}
template <int V>
__device__ __forceinline__ void store(void* p, bool bf16, int64_t i, const float (&v)[V]) {
  if constexpr (V == 4) {
    if (bf16)
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + i) =
          make_uint2(to_bf16(v[0]) | to_bf16(v[1]) << 16, to_bf16(v[2]) | to_bf16(v[3]) << 16);
    else
      *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else if (bf16) {
    static_cast<uint16_t*>(p)[i] = (uint16_t)to_bf16(v[0]);
  } else {
    static_cast<float*>(p)[i] = v[0];
  }
}

// Sum over the T threads of a row; the same value in all of them.
template <int T>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (T > 64) {
    __syncthreads();   // the last sum's readers are done
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) v += part[w];
  }
  return v;
}

// T threads a row, each of them E pieces of V elements.
template <int T, int E, int V>
struct Row {
  float v[E][V];
  int D, t;
  template <class F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = (e * T + t) * V;
      if (i < D) f(e, i);
    }
  }
  // v becomes norm(v)
  __device__ __forceinline__ void norm(int kind, float eps, const float* gamma, const float* beta, float* part) {
    float mean = 0.0f;
    if (kind == C4S_NORM_LAYER) {
      float s = 0.0f;
      each([&](int e, int) {
#pragma unroll
        for (int j = 0; j < V; ++j) s += v[e][j];
      });
      mean = row_sum<T>(s, part) / (float)D;
    }
    float q = 0.0f;
    each([&](int e, int) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[e][j] -= mean;
        q = __builtin_fmaf(v[e][j], v[e][j], q);
      }
    });
    const float inv = 1.0f / sqrtf(row_sum<T>(q, part) / (float)D + eps);
    each([&](int e, int i) {
      float g[V], b[V];
#pragma unroll
      for (int j = 0; j < V; ++j) { g[j] = 1.0f; b[j] = 0.0f; }
      if (gamma) load<V>(gamma, false, i, g);
      if (beta) load<V>(beta, false, i, b);
#pragma unroll
      for (int j = 0; j < V; ++j) v[e][j] = __builtin_fmaf(v[e][j] * inv, g[j], b[j]);
    });
  }
};

constexpr int kNormThreads = 256;

template <int T, int E, int V>
__global__ __launch_bounds__(T > kNormThreads ? T : kNormThreads) void k_block_norm(c4s_norm a) {
  constexpr int kRows = T < kNormThreads ? kNormThreads / T : 1;
  __shared__ float part[16];
  const int m = blockIdx.x * kRows + (kRows > 1 ? (int)threadIdx.x / T : 0);
  if (m >= a.M) return;   // whole waves: with T > 64 a workgroup is one row
  const bool xb = a.x_dtype == C4S_DTYPE_BF16;
  Row<T, E, V> r;
  r.D = a.D;
  r.t = threadIdx.x % T;
  const int64_t x0 = (int64_t)m * a.ldx;
  if (a.y) {
    const bool yb = a.y_dtype == C4S_DTYPE_BF16;
    const int64_t y0 = (int64_t)m * a.ldy;
    float x[E][V];
    r.each([&](int e, int i) { load<V>(a.x, xb, x0 + i, x[e]); });
    r.each([&](int e, int i) { load<V>(a.y, yb, y0 + i, r.v[e]); });
    if (a.post) r.norm(a.kind, a.eps, a.post_gamma, a.post_beta, part);
    const int64_t g0 = a.gate ? (int64_t)(m / a.gate_rows) * a.ld_gate : 0;
    r.each([&](int e, int i) {
      float g[V];
#pragma unroll
      for (int j = 0; j < V; ++j) g[j] = 1.0f;
      if (a.gate) load<V>(a.gate, false, g0 + i, g);
#pragma unroll
      for (int j = 0; j < V; ++j) r.v[e][j] = __builtin_fmaf(a.res_scale * g[j], r.v[e][j], x[e][j]);
    });
  } else {
    r.each([&](int e, int i) { load<V>(a.x, xb, x0 + i, r.v[e]); });
  }
  if (a.x_out) r.each([&](int e, int i) { store<V>(a.x_out, xb, (int64_t)m * a.ld_x_out + i, r.v[e]); });
  if (!a.out) return;
  r.norm(a.kind, a.eps, a.gamma, a.beta, part);
  r.each([&](int e, int i) { store<V>(a.out, a.out_dtype == C4S_DTYPE_BF16, (int64_t)m * a.ld_out + i, r.v[e]); });
}

template <int T, int E, int V>
hipError_t launch(const c4s_norm& a, hipStream_t s) {
  constexpr int kRows = T < kNormThreads ? kNormThreads / T : 1;
  hipLaunchKernelGGL((k_block_norm<T, E, V>), dim3((a.M + kRows - 1) / kRows), dim3(T > kNormThreads ? T : kNormThreads), 0, s, a);
  return hipGetLastError();
}

// Whether every row of a tensor can be read four elements at a time.
bool by_four(const void* p, int64_t ld, int32_t dtype) {
  return !p || (ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (dtype == C4S_DTYPE_BF16 ? 8 : 16) == 0);
}

__global__ void k_zero(uint32_t* p, size_t n) {
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0u;
}

}  // namespace

hipError_t launch_zero(void* p, size_t bytes, hipStream_t s) {
  hipLaunchKernelGGL(k_zero, dim3(64), dim3(256), 0, s, static_cast<uint32_t*>(p), bytes / 4);
  return hipGetLastError();
}

hipError_t launch_block_norm(const c4s_norm& a, hipStream_t s) {
  const bool four = a.D % 4 == 0 && by_four(a.x, a.ldx, a.x_dtype) && by_four(a.y, a.ldy, a.y_dtype) &&
                    by_four(a.x_out, a.ld_x_out, a.x_dtype) && by_four(a.out, a.ld_out, a.out_dtype) &&
                    by_four(a.gate, a.ld_gate, C4S_DTYPE_F32) && by_four(a.gamma, 0, C4S_DTYPE_F32) &&
                    by_four(a.beta, 0, C4S_DTYPE_F32) && by_four(a.post_gamma, 0, C4S_DTYPE_F32) &&
                    by_four(a.post_beta, 0, C4S_DTYPE_F32);
  if (four) {
    if (a.D <= 2048) return launch<64, 8, 4>(a, s);
    if (a.D <= 8192) return launch<256, 8, 4>(a, s);
    return launch<1024, 4, 4>(a, s);
  }
  if (a.D <= 1024) return launch<64, 16, 1>(a, s);
  if (a.D <= 4096) return launch<256, 16, 1>(a, s);
  return launch<1024, 16, 1>(a, s);
}

}  // namespace c4s
