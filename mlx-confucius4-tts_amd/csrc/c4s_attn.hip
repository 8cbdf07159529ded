// Attention of new tokens over the paged cache (c4s_attn, include/c4s_layers.h).
//
// A workgroup has 16 rows (token, query head) of one sequence and key head; its
// waves take blocks of 64 positions in turn, each with a running maximum and
// sum of its own, and are joined at the end in LDS.
//
// Both products run transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane
// always holds one row (column l % 16 of the results): the maximum, the sum and
// the rescaling are a lane's own, but for two steps across the four lanes that
// share a row. Which positions of the block a matrix row of S^T stands for is
// free; row 4 g + i of tile t is position 16 g + 4 t + i, so that lane group g
// ends up with the weights of positions 16 g .. 16 g + 15, which is what P^T wants
// of it as the next product's operand, and which lie next to each other in a
// page of the values. Nothing is shuffled or transposed in between, and keys
// and values go from memory straight into the matrix engine's registers.
//
// The weights enter the second product as bf16 pairs (hi + lo, about 2^-17
// relative): rounded once to bf16 they would add an error of the size of the
// output's own rounding.

#include <hip/hip_runtime.h>

#include "c4s_layers.hpp"

namespace c4s {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));
}
__device__ __forceinline__ float low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// Eight int8 codes as bf16 (exact).
__device__ __forceinline__ uint4 codes(uint2 q) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? q.x : q.y;
    const float a = (float)(int8_t)(w >> (16 * (i & 1))), b = (float)(int8_t)(w >> (16 * (i & 1) + 8));
    o[i] = (__float_as_uint(a) >> 16) | (__float_as_uint(b) & 0xFFFF0000u);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Over the four lanes that share a row.
__device__ __forceinline__ float max4(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float sum4(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// Dwords of two bf16, of which those at index lo .. hi - 1 stay and the others become zero.
__device__ __forceinline__ uint4 keep(uint4 w, int at, int lo, int hi) {
  uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = at + 2 * i;
    v[i] &= (j >= lo && j < hi ? 0xFFFFu : 0u) | (j + 1 >= lo && j + 1 < hi ? 0xFFFF0000u : 0u);
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ bool odd_exp(uint32_t w) {   // either half inf or NaN
  return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}

// The finite halves of w, and ones where the others were.
__device__ __forceinline__ void part_odd(uint32_t& w, uint32_t& odd) {
  odd = ((w & 0x7F80u) == 0x7F80u ? 0x3F80u : 0u) | ((w & 0x7F800000u) == 0x7F800000u ? 0x3F800000u : 0u);
  w &= (odd & 0xFFFFu ? 0u : 0xFFFFu) | (odd >> 16 ? 0u : 0xFFFF0000u);
}

constexpr int kRows = 16;
constexpr int kKeys = 64;    // positions a wave takes at a time
constexpr int kWaves = 4;
constexpr int kAttnThreads = 64 * kWaves;

// DH: the head's dims rounded up to 64, 128 or 256.
template <int DH, bool Q8>
__global__ __launch_bounds__(kAttnThreads) void k_attn(AttnArgs a) {
  constexpr int kSteps = DH / 32, kTiles = DH / 16;
  __shared__ float sm[kWaves][kRows], sl[kWaves][kRows];
  __shared__ __align__(16) float so[kWaves - 1][kRows][DH + 4];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, g = lane / 16;
  const int head = blockIdx.x % a.c.n_heads, seq = blockIdx.y, dim = a.c.dim;
  int row0 = seq, n_new = 1;
  if (a.off) {
    row0 = a.off[seq];
    const int end = min(a.off[seq + 1], a.n_rows);
    if (row0 < 0) return;
    n_new = min(end - row0, a.max_new);
  } else if (seq >= a.n_rows) {
    return;
  }
  const int n_all = n_new * a.shared, r0 = blockIdx.x / a.c.n_heads * kRows;
  if (r0 >= n_all) return;
  const int len = a.lens[seq];
  const int past = len - (a.off ? a.off[seq + 1] - row0 : 1);
  const int cap = a.c.max_pages << a.c.page_shift;
  const int fst = a.first ? min(max(a.first[seq], 0), cap) : 0;
  // lane's row
  const int r = min(r0 + c, n_all - 1);
  const int token = r / a.shared, qh = head * a.shared + r % a.shared;
  const int lim = min(past + token + 1, cap);           // positions this row sees end here
  const int least = min(past + r0 / a.shared + 1, cap);   // ... the tile's first row
  const int kend = min(past + min(r0 + kRows - 1, n_all - 1) / a.shared + 1, cap);

  uint4 q[kSteps];
  const uint16_t* qp = a.q + (int64_t)(row0 + token) * a.ldq + qh * dim;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    // codes come 16 dims a lane at a time, which are two steps of 8
    const int d = Q8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
    q[s] = d < dim ? *reinterpret_cast<const uint4*>(qp + d) : make_uint4(0, 0, 0, 0);
  }

  const float c2 = a.scale * kLog2e;
  float m = -__builtin_inff(), l = 0.0f;
  f32x4 o[kTiles] = {};
  const int ps = 1 << a.c.page_shift;
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_ld;
  const int64_t page_elems = (int64_t)ps * dim;

  for (int t = (fst & ~(kKeys - 1)) + wave * kKeys; t < kend; t += kWaves * kKeys) {
    // pages of the key row this lane loads, and of the 16 positions it weighs
    const int kt = t + 16 * (c / 4), vt = t + 16 * g;
    int kp = -1, vp = -1;
    if ((kt >> a.c.page_shift) < a.c.max_pages) kp = table[kt >> a.c.page_shift];
    if ((vt >> a.c.page_shift) < a.c.max_pages) vp = table[vt >> a.c.page_shift];
    const bool there = vp >= 0 && vp < a.c.n_pages;
    if (kp < 0 || kp >= a.c.n_pages) kp = 0;   // its scores are dropped
    if (!there) vp = 0;
    const int64_t kb = ((int64_t)kp * a.c.n_heads + head) * page_elems + (int64_t)((kt & (ps - 1)) + c % 4) * dim;
    const int64_t vslot = ((int64_t)vp * a.c.n_heads + head) * ps + (vt & (ps - 1));
    const int64_t vb = vslot * dim - (int64_t)(vt & (ps - 1)) * dim + (vt & (ps - 1));

    f32x4 s[4] = {};
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      if constexpr (Q8) {
        const uint8_t* k = static_cast<const uint8_t*>(a.c.k) + kb + (int64_t)(4 * tt) * dim;
#pragma unroll
        for (int st = 0; st < kSteps; st += 2) {
          const int d = 32 * st + 16 * g;
          const uint4 w = d < dim ? *reinterpret_cast<const uint4*>(k + d) : make_uint4(0, 0, 0, 0);
          s[tt] = mfma(codes(make_uint2(w.x, w.y)), q[st], s[tt]);
          s[tt] = mfma(codes(make_uint2(w.z, w.w)), q[st + 1], s[tt]);
        }
      } else {
        const uint16_t* k = static_cast<const uint16_t*>(a.c.k) + kb + (int64_t)(4 * tt) * dim;
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          const int d = 32 * st + 8 * g;
          s[tt] = mfma(d < dim ? *reinterpret_cast<const uint4*>(k + d) : make_uint4(0, 0, 0, 0), q[st], s[tt]);
        }
      }
    }
    // lane's 16 scores are positions vt .. vt + 15 of its row, in order
    float p[16], vs[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      float f = c2;
      if constexpr (Q8) f *= a.c.k_scale[vslot + j];
      p[j] = s[j / 4][j % 4] * f;
      if constexpr (Q8) vs[j] = a.c.v_scale[vslot + j];
    }
    const bool edge = t < fst || t + kKeys > least || __any(!there);
    if (edge) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (!there || vt + j < fst || vt + j >= lim) p[j] = -__builtin_inff();
    }
    float top = p[0];
#pragma unroll
    for (int j = 1; j < 16; ++j) top = fmaxf(top, p[j]);
    top = fmaxf(max4(top), m);
    const float base = top == -__builtin_inff() ? 0.0f : top;   // nothing seen yet
    const float old = exp2f(m - base);
    m = top;
    l *= old;
#pragma unroll
    for (int d = 0; d < kTiles; ++d) o[d] *= old;
    uint32_t hi[8], lo[8];
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
      float x = exp2f(p[j] - base), y = exp2f(p[j + 1] - base);
      l += x + y;
      if constexpr (Q8) {   // 0 for a masked position, whatever its scale
        x = x != 0.0f ? x * vs[j] : 0.0f;
        y = y != 0.0f ? y * vs[j + 1] : 0.0f;
      }
      hi[j / 2] = pack(x, y);
      lo[j / 2] = pack(x - low(hi[j / 2]), y - high(hi[j / 2]));
    }
    const int from = there ? fst - vt : 16, to = there ? kend - vt : 16;
#pragma unroll
    for (int d = 0; d < kTiles; ++d) {
      if (16 * d >= dim) break;
      uint4 v[2];
      if constexpr (Q8) {
        const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.c.v) + vb + (int64_t)(16 * d + c) * ps);
        v[0] = codes(make_uint2(w.x, w.y));
        v[1] = codes(make_uint2(w.z, w.w));
      } else {
        const uint16_t* vr = static_cast<const uint16_t*>(a.c.v) + vb + (int64_t)(16 * d + c) * ps;
        v[0] = *reinterpret_cast<const uint4*>(vr);
        v[1] = *reinterpret_cast<const uint4*>(vr + 8);
        if (edge) {
          v[0] = keep(v[0], 0, from, to);
          v[1] = keep(v[1], 8, from, to);
          // A value that is not finite, in a block that some rows see in part:
          // 0 times it would reach the rows that do not see it.
          uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w}, odd[8];
          bool any = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) any = any || odd_exp(w[i]);
          if (__any(any)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) part_odd(w[i], odd[i]);
            f32x4 seen = {};
#pragma unroll
            for (int st = 0; st < 2; ++st) {
              v[st] = make_uint4(w[4 * st], w[4 * st + 1], w[4 * st + 2], w[4 * st + 3]);
              seen = mfma(make_uint4(odd[4 * st], odd[4 * st + 1], odd[4 * st + 2], odd[4 * st + 3]),
                          make_uint4(hi[4 * st], hi[4 * st + 1], hi[4 * st + 2], hi[4 * st + 3]), seen);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (seen[i] != 0.0f) o[d][i] = __builtin_nanf("");
          }
        }
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        o[d] = mfma(v[st], make_uint4(hi[4 * st], hi[4 * st + 1], hi[4 * st + 2], hi[4 * st + 3]), o[d]);
        o[d] = mfma(v[st], make_uint4(lo[4 * st], lo[4 * st + 1], lo[4 * st + 2], lo[4 * st + 3]), o[d]);
      }
    }
  }

  // the waves' parts, joined by wave 0
  l = sum4(l);
  if (g == 0) {
    sm[wave][c] = m;
    sl[wave][c] = l;
  }
  if (wave > 0) {
#pragma unroll
    for (int d = 0; d < kTiles; ++d) *reinterpret_cast<f32x4*>(&so[wave - 1][c][16 * d + 4 * g]) = o[d];
  }
  __syncthreads();
  if (wave > 0 || r0 + c >= n_all) return;
  float top = m;
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, sm[w][c]);
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float f[kWaves], sum = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    f[w] = exp2f(sm[w][c] - base);
    sum += sl[w][c] * f[w];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  uint16_t* out = a.out + (int64_t)(row0 + token) * a.ld_out + qh * dim;
#pragma unroll
  for (int d = 0; d < kTiles; ++d) {
    if (16 * d >= dim) break;
    f32x4 v = o[d] * f[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(&so[w - 1][c][16 * d + 4 * g]);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(x[i], f[w], v[i]);
    }
    *reinterpret_cast<uint2*>(out + 16 * d + 4 * g) = make_uint2(pack(v[0] * inv, v[1] * inv), pack(v[2] * inv, v[3] * inv));
  }
  if (a.lse && g == 0)
    a.lse[(int64_t)(row0 + token) * a.n_heads + qh] = sum == 0.0f ? -__builtin_inff() : (top + log2f(sum)) * kLn2;
}

}  // namespace

hipError_t launch_attn(const AttnArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(((int64_t)a.max_new * a.shared + kRows - 1) / kRows * a.c.n_heads), a.c.n_seqs);
  const bool q8 = a.c.store == C4S_KV_Q8;
  if (a.c.dim <= 64) {
    if (q8) hipLaunchKernelGGL((k_attn<64, true>), grid, dim3(kAttnThreads), 0, s, a);
    else hipLaunchKernelGGL((k_attn<64, false>), grid, dim3(kAttnThreads), 0, s, a);
  } else if (a.c.dim <= 128) {
    if (q8) hipLaunchKernelGGL((k_attn<128, true>), grid, dim3(kAttnThreads), 0, s, a);
    else hipLaunchKernelGGL((k_attn<128, false>), grid, dim3(kAttnThreads), 0, s, a);
  } else {
    if (q8) hipLaunchKernelGGL((k_attn<256, true>), grid, dim3(kAttnThreads), 0, s, a);
    else hipLaunchKernelGGL((k_attn<256, false>), grid, dim3(kAttnThreads), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace c4s
