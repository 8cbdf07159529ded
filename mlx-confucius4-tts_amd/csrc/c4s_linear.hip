// Product with bias, activation and residual in its epilogue (c4s_linear,
// include/c4s_layers.h), bf16 activations, weights in bf16 or 8-bit codes.
//
// v_mfma_f32_16x16x32_bf16 with the weights as its rows (A: lane l holds row
// l % 16, inputs (l / 16) 8 .. + 7) and the activations as its columns (B the
// same way): a lane's four results are four consecutive outputs of one row, so
// the epilogue loads and stores vectors.
//
// 8-bit codes go into the matrix engine as q - 128, which bf16 holds exactly:
//   sum_k x w = sum_g s_g P_g + (b_g + 128 s_g) X_g,
// P_g = sum_{k in g} x (q - 128) and X_g = sum_{k in g} x, both exact products
// summed in fp32, X_g as a product with ones. Nothing is rounded that the codes
// themselves do not round.

#include <hip/hip_runtime.h>

#include "c4s_layers.hpp"

namespace c4s {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float from_bf16(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

// Eight codes as bf16 q - 128 (exact).
__device__ __forceinline__ uint4 centred(uint2 q) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = (i < 2 ? q.x : q.y) >> (16 * (i & 1));
    const float lo = (float)(w & 0xFFu) - 128.0f, hi = (float)((w >> 8) & 0xFFu) - 128.0f;
    o[i] = (__float_as_uint(lo) >> 16) | (__float_as_uint(hi) & 0xFFFF0000u);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

__device__ __forceinline__ float activate(float y, int act) {
  if (act == C4S_ACT_GELU) {   // y / 2 (1 + tanh u) = y / (1 + exp(-2 u))
    const float u = 0.7978845608028654f * __builtin_fmaf(0.044715f * y * y, y, y);
    return y / (1.0f + expf(-2.0f * u));
  }
  if (act == C4S_ACT_SILU) return y / (1.0f + expf(-y));
  if (act == C4S_ACT_RELU) return y > 0.0f ? y : (y != y ? y : 0.0f);
  return y;
}

// Four consecutive outputs n .. n + 3 of row m: bias, activation, residual, store.
__device__ __forceinline__ void finish(const c4s_linear_desc& a, int m, int n, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.N) break;
    float y = acc[i] + (a.bias ? a.bias[n + i] : 0.0f);
    y = activate(y, a.act);
    if (a.residual) {
      const int64_t o = (int64_t)m * a.ld_res + n + i;
      y += a.res_dtype == C4S_DTYPE_BF16 ? from_bf16(static_cast<const uint16_t*>(a.residual)[o]) : static_cast<const float*>(a.residual)[o];
    }
    const int64_t o = (int64_t)m * a.ld_out + n + i;
    if (a.out_dtype == C4S_DTYPE_BF16) static_cast<uint16_t*>(a.out)[o] = (uint16_t)to_bf16(y);
    else static_cast<float*>(a.out)[o] = y;
  }
}

constexpr int kThreads = 256;
constexpr int kMB = 4;   // 16-row blocks of activations a workgroup takes

// Each wave 16 outputs of up to 64 rows, everything straight from memory.
template <bool Q8>
__global__ __launch_bounds__(kThreads) void k_linear(c4s_linear_desc a) {
  const int lane = threadIdx.x % 64, c = lane % 16, g = lane / 16;
  const int n0 = (blockIdx.y * (kThreads / 64) + threadIdx.x / 64) * 16, m0 = blockIdx.x * 16 * kMB;
  if (n0 >= a.N) return;
  const int n = min(n0 + c, a.N - 1);
  const uint16_t* x[kMB];
#pragma unroll
  for (int b = 0; b < kMB; ++b) x[b] = a.x + (int64_t)min(m0 + 16 * b + c, a.M - 1) * a.ldx;
  f32x4 acc[kMB] = {};
  const int step = Q8 ? a.group : 32;
  for (int k0 = 0; k0 < a.K; k0 += step) {
    f32x4 part[kMB] = {}, sum[kMB] = {};
    for (int k = k0 + 8 * g; k < k0 + step; k += 32) {
      uint4 w = make_uint4(0, 0, 0, 0), xv[kMB];
      if (k < a.K) {
        if constexpr (Q8) w = centred(*reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.weight) + (int64_t)n * a.K + k));
        else w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.weight) + (int64_t)n * a.K + k);
      }
#pragma unroll
      for (int b = 0; b < kMB; ++b) {
        xv[b] = make_uint4(0, 0, 0, 0);
        if (k < a.K) xv[b] = *reinterpret_cast<const uint4*>(x[b] + k);
        if constexpr (Q8) {
          const uint32_t one = 0x3F803F80u;
          part[b] = mfma(w, xv[b], part[b]);
          sum[b] = mfma(make_uint4(one, one, one, one), xv[b], sum[b]);
        } else {
          acc[b] = mfma(w, xv[b], acc[b]);
        }
      }
    }
    if constexpr (Q8) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t o = (int64_t)min(n0 + 4 * g + i, a.N - 1) * (a.K / a.group) + k0 / a.group;
        const float s = a.wscale[o], off = __builtin_fmaf(128.0f, s, a.wbias[o]);
#pragma unroll
        for (int b = 0; b < kMB; ++b) acc[b][i] = __builtin_fmaf(s, part[b][i], __builtin_fmaf(off, sum[b][i], acc[b][i]));
      }
    }
  }
#pragma unroll
  for (int b = 0; b < kMB; ++b) {
    const int m = m0 + 16 * b + c;
    if (m < a.M) finish(a, m, n0 + 4 * g, acc[b]);
  }
}

}  // namespace

hipError_t launch_linear(const c4s_linear_desc& a, hipStream_t s) {
  const dim3 grid((a.M + 16 * kMB - 1) / (16 * kMB), (a.N + 63) / 64);
  if (a.wdtype == C4S_W_Q8) hipLaunchKernelGGL(k_linear<true>, grid, dim3(kThreads), 0, s, a);
  else hipLaunchKernelGGL(k_linear<false>, grid, dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace c4s
