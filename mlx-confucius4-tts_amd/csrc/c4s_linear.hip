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

#include "c4s_join.hpp"
#include "c4s_layers.hpp"

namespace c4s {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 Quad __attribute__((ext_vector_type(4)));   // these round to nearest even
typedef __bf16 Pair __attribute__((ext_vector_type(2)));
typedef uint32_t Eight __attribute__((ext_vector_type(4), aligned(8)));   // eight bf16

__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ float from_bf16(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t to_bf16(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }

// A tile's rows behind a buffer descriptor: offsets are 32 bits from its first
// row, and rows behind the last read as zeros.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
struct Tile {
  u32x4 d;
  // `rows` rows of `width` bytes, `pitch` bytes apart, from p on: up to 2^31 bytes.
  __device__ __forceinline__ Tile(const void* p, int64_t rows, uint32_t width, uint32_t pitch) {
    const uint64_t b = reinterpret_cast<uint64_t>(p);
    d = u32x4{(uint32_t)b, (uint32_t)(b >> 32) & 0xFFFFu, (uint32_t)((rows - 1) * pitch + width), 0x00027000u};
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)d[1] << 32 | d[0]), 0, (int)d[2], (int)d[3]);
  }
  // 16 (8) bytes at v. (The whole offset is the lane's own: the instruction's
  // scalar offset is not part of the bounds check.)
  __device__ __forceinline__ uint4 load(uint32_t v) const {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rsrc(), (int)v, 0, 0));
  }
  __device__ __forceinline__ uint2 load8(uint32_t v) const {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rsrc(), (int)v, 0, 0));
  }
};

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

// y / (1 + 2^z): the exponential and the reciprocal as the hardware has them (an
// ulp each; an infinite 2^z gives 0 y).
__device__ __forceinline__ float sigmoid_of(float y, float z) {
  return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z));
}
template <int N>
__device__ __forceinline__ void activate(float (&y)[N], int act) {
  if (act == C4S_ACT_GELU) {   // y / 2 (1 + tanh u) = y / (1 + exp(-2 u)), u = sqrt(2 / pi) (y + 0.044715 y^3)
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = sigmoid_of(y[i], y[i] * __builtin_fmaf(-0.10294324f, y[i] * y[i], -2.3022082f));
  } else if (act == C4S_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = sigmoid_of(y[i], y[i] * -1.4426950408889634f);
  } else if (act == C4S_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = y[i] > 0.0f ? y[i] : (y[i] != y[i] ? y[i] : 0.0f);
  }
}

// Four values of the residual, from element o on.
__device__ __forceinline__ f32x4 residual4(const c4s_linear_desc& a, int64_t o) {
  if (a.res_dtype != C4S_DTYPE_BF16) return *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.residual) + o);
  const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.residual) + o);
  return f32x4{from_bf16(w.x & 0xFFFFu), from_bf16(w.x >> 16), from_bf16(w.y & 0xFFFFu), from_bf16(w.y >> 16)};
}

// Four consecutive outputs n .. n + 3 of row m: bias, activation, residual, store.
// Few: n + 3 may lie behind the last output, or the tensors' rows off four elements' alignment.
__device__ __forceinline__ void finish(const c4s_linear_desc& a, bool vec, int m, int n, f32x4 y) {
  if (!vec) {
#pragma unroll 1
    for (int i = 0; i < 4 && n + i < a.N; ++i) {
      float u[1] = {(i < 2 ? (i ? y[1] : y[0]) : (i > 2 ? y[3] : y[2])) + (a.bias ? a.bias[n + i] : 0.0f)};
      activate(u, a.act);
      float v = u[0];
      const int64_t r = (int64_t)m * a.ld_res + n + i, o = (int64_t)m * a.ld_out + n + i;
      if (a.residual)
        v += a.res_dtype == C4S_DTYPE_BF16 ? from_bf16(static_cast<const uint16_t*>(a.residual)[r]) : static_cast<const float*>(a.residual)[r];
      if (a.out_dtype == C4S_DTYPE_BF16) static_cast<uint16_t*>(a.out)[o] = (uint16_t)to_bf16(v);
      else static_cast<float*>(a.out)[o] = v;
    }
    return;
  }
  if (n >= a.N) return;
  f32x4 b = {};
  if (a.bias) b = *reinterpret_cast<const f32x4*>(a.bias + n);
  float v[4] = {y[0] + b[0], y[1] + b[1], y[2] + b[2], y[3] + b[3]};
  activate(v, a.act);
  y = f32x4{v[0], v[1], v[2], v[3]};
  if (a.residual) y += residual4(a, (int64_t)m * a.ld_res + n);
  const int64_t o = (int64_t)m * a.ld_out + n;
  if (a.out_dtype == C4S_DTYPE_BF16)
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + o) = __builtin_bit_cast(uint2, Quad{(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]});
  else
    *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + o) = y;
}

// Whether finish() may use vectors.
bool vectors(const c4s_linear_desc& a) {
  auto four = [](const void* p, int64_t ld, int32_t dtype) {
    return !p || (ld % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (dtype == C4S_DTYPE_BF16 ? 8 : 16) == 0);
  };
  return a.N % 4 == 0 && four(a.out, a.ld_out, a.out_dtype) && four(a.residual, a.ld_res, a.res_dtype) && four(a.bias, 0, C4S_DTYPE_F32);
}

// ---- few rows ---------------------------------------------------------------------------
//
// Up to 64 rows a tile: the weights' bytes are what it costs, so they pass once
// and everything else makes room for their loads. A workgroup has 32 outputs
// and a slice of K; its waves (W, 4 or 8) take the slice's chunks of 64 inputs in turn,
// each on its own: a chunk's rows (of the weights and of the activations, 128
// bytes a row) are loaded whole lines at a time, one chunk ahead, into
// registers, and pass through the wave's part of LDS into fragment order, with
// no barrier before the waves' sums are joined at the end. (Fragments straight
// from memory are 16 rows of 64 bytes a load; with rows K apart they fall into
// few sets of the L1: 64 x 1280 x 5120 took 165 us that way.)
//
// Where the outputs alone give too few workgroups (few_splits), K is split over
// several, which leave their sums in the workspace; the last to arrive adds
// them in the order of the slices, so that the result does not depend on it.
constexpr int kFewN = 32;
constexpr int kFewM = 64;
constexpr int kChunk = 64;

struct FewArgs {
  c4s_linear_desc d;
  bool vec;
  int splits, n_tiles;
  uint32_t* arrived;   // [tiles], zero between calls
  float* part;         // [tiles][splits][kFewM][kFewN]
};

// Byte offset of 16-byte piece p of row r in a wave's LDS: rows of 8 pieces, the
// pieces permuted so that 16 rows' reads of one piece fall into different banks.
__device__ __forceinline__ int piece(int r, int p) { return r * 128 + ((p ^ ((r >> 1) & 7)) << 4); }

template <bool Q8, int MB>
struct FewChunk {   // a chunk's loads in flight
  uint4 x[2 * MB];          // rows 8 j + lane / 8, piece lane % 8
  uint4 w[Q8 ? 2 : 4];      // bf16: the same of the weights; codes: rows 16 j + lane / 4, 16 codes
  float s[2];               // scales (lanes 0 .. 31) and offsets (32 .. 63) of the chunk's two halves
};

template <bool Q8, int MB, int W>
__global__ __launch_bounds__(64 * W, W == 4 ? 2 : 1) void k_linear_few(FewArgs f) {
  constexpr int kXBytes = 16 * MB * 128, kWBytes = kFewN * 128, kSBytes = Q8 ? 512 : 0;
  constexpr int kWaveBytes = kXBytes + kWBytes + kSBytes, kPitch = kFewN + 4;
  constexpr int kRedBytes = W * 16 * MB * kPitch * 4;
  __shared__ __align__(16) char lds[W * kWaveBytes > kRedBytes ? W * kWaveBytes : kRedBytes];
  const c4s_linear_desc& a = f.d;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, c = lane % 16, g = lane / 16;
  const int tile = blockIdx.x / f.splits, split = blockIdx.x % f.splits;
  const int n0 = tile % f.n_tiles * kFewN, m0 = tile / f.n_tiles * kFewM;
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const int c0 = (int)((int64_t)chunks * split / f.splits), c1 = (int)((int64_t)chunks * (split + 1) / f.splits);

  constexpr int kWSize = Q8 ? 1 : 2;   // bytes a weight
  const uint32_t xp = 2u * (uint32_t)a.ldx, wp = (uint32_t)kWSize * (uint32_t)a.K;   // rows apart
  const Tile xt(a.x + (int64_t)m0 * a.ldx, min(a.M - m0, 16 * MB), 2u * a.K, xp);
  const Tile wt(static_cast<const char*>(a.weight) + (int64_t)n0 * wp, min(a.N - n0, kFewN), wp, wp);
  const uint32_t xo = lane / 8 * xp + lane % 8 * 16, wo = Q8 ? lane / 4 * wp + lane % 4 * 16 : lane / 8 * wp + lane % 8 * 16;
  const float* sr = nullptr;
  int half = 1;   // groups that start in the second half of a chunk: of 32 inputs, else the chunk's own
  if constexpr (Q8) {
    const int groups = a.K / a.group;
    sr = (lane < 32 ? a.wscale : a.wbias) + (int64_t)min(n0 + lane % 32, a.N - 1) * groups;
    half = a.group == 32 ? 1 : 0;
  }
  // Inputs behind the last are the next row's first, or zeros; stage() drops them.
  auto load = [&](FewChunk<Q8, MB>& r, int ch) {
    const int k0 = ch * kChunk;
#pragma unroll
    for (int j = 0; j < 2 * MB; ++j) r.x[j] = xt.load(xo + 8 * j * xp + 2 * k0);
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {   // codes are aligned to 8 bytes
        const uint2 lo = wt.load8(wo + 16 * j * wp + k0), hi = wt.load8(wo + 16 * j * wp + k0 + 8);
        r.w[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
      const int gi = k0 / a.group;
      r.s[0] = sr[gi];
      r.s[1] = sr[min(gi + half, a.K / a.group - 1)];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[j] = wt.load(wo + 8 * j * wp + 2 * k0);
    }
  };
  char* xs = lds + wave * kWaveBytes;
  char* ws = xs + kXBytes;
  f32x4 acc[2][MB] = {};
  auto stage = [&](FewChunk<Q8, MB>& r, int ch) {
    // (codes are finite whatever they are: zeros on the other side do)
    if (ch * kChunk + kChunk > a.K && ch * kChunk + lane % 8 * 8 >= a.K) {
#pragma unroll
      for (int j = 0; j < 2 * MB; ++j) r.x[j] = make_uint4(0, 0, 0, 0);
      if constexpr (!Q8)
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[j] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 2 * MB; ++j) *reinterpret_cast<uint4*>(xs + piece(8 * j + lane / 8, lane % 8)) = r.x[j];
    if constexpr (Q8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) *reinterpret_cast<uint4*>(ws + (16 * j + lane / 4) * 80 + lane % 4 * 16) = r.w[j];
      float* sp = reinterpret_cast<float*>(ws + kWBytes);
      sp[lane] = r.s[0];
      sp[64 + lane] = r.s[1];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(ws + piece(8 * j + lane / 8, lane % 8)) = r.w[j];
    }
  };
  auto compute = [&] {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint4 xv[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) xv[b] = *reinterpret_cast<const uint4*>(xs + piece(16 * b + c, 4 * st + g));
      if constexpr (Q8) {
        const float* sp = reinterpret_cast<const float*>(ws + kWBytes) + 64 * st;
        const uint32_t one = 0x3F803F80u;
        f32x4 sum[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) sum[b] = mfma(make_uint4(one, one, one, one), xv[b], f32x4{});
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          const uint4 w = centred(*reinterpret_cast<const uint2*>(ws + (16 * nb + c) * 80 + 32 * st + 8 * g));
          const f32x4 s = *reinterpret_cast<const f32x4*>(sp + 16 * nb + 4 * g), o = *reinterpret_cast<const f32x4*>(sp + 32 + 16 * nb + 4 * g);
#pragma unroll
          for (int b = 0; b < MB; ++b) {
            const f32x4 p = mfma(w, xv[b], f32x4{});
#pragma unroll
            for (int i = 0; i < 4; ++i)
              acc[nb][b][i] = __builtin_fmaf(s[i], p[i], __builtin_fmaf(__builtin_fmaf(128.0f, s[i], o[i]), sum[b][i], acc[nb][b][i]));
          }
        }
      } else {
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
          const uint4 w = *reinterpret_cast<const uint4*>(ws + piece(16 * nb + c, 4 * st + g));
#pragma unroll
          for (int b = 0; b < MB; ++b) acc[nb][b] = mfma(w, xv[b], acc[nb][b]);
        }
      }
    }
  };
  FewChunk<Q8, MB> r;
  int ch = c0 + wave;
  if (ch < c1) load(r, ch);
  // Lanes of the wave read what others wrote: order that the compiler keeps (it costs no instruction; LDS serves a
  // wave's accesses in order).
  auto wave_order = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  for (; ch < c1; ch += W) {
    stage(r, ch);
    wave_order();
    if (ch + W < c1) load(r, ch + W);
    compute();
    wave_order();
  }

  // the waves' sums
  __syncthreads();
  float* red = reinterpret_cast<float*>(lds);
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int b = 0; b < MB; ++b)
      *reinterpret_cast<f32x4*>(red + (wave * 16 * MB + 16 * b + c) * kPitch + 16 * nb + 4 * g) = acc[nb][b];
  __syncthreads();
  constexpr int kQuads = 16 * MB * kFewN / 4;   // of four outputs
  const int rows = min(16 * MB, a.M - m0);
#pragma unroll
  for (int i = 0; i < (kQuads + (64 * W) - 1) / (64 * W); ++i) {
    const int q = threadIdx.x + i * (64 * W), m = q / (kFewN / 4), n = q % (kFewN / 4) * 4;
    if (q >= kQuads || m >= rows) continue;
    f32x4 y = *reinterpret_cast<const f32x4*>(red + m * kPitch + n);
#pragma unroll
    for (int w = 1; w < W; ++w) y += *reinterpret_cast<const f32x4*>(red + (w * 16 * MB + m) * kPitch + n);
    if (f.splits == 1) finish(a, f.vec, m0 + m, n0 + n, y);
    else put_quad(f.part + (int64_t)blockIdx.x * kFewM * kFewN, kQuads, q, y);
  }
  if (f.splits == 1 || !last_to_arrive(f.arrived + tile, f.splits)) return;
#pragma unroll
  for (int i = 0; i < (kQuads + (64 * W) - 1) / (64 * W); ++i) {
    const int q = threadIdx.x + i * (64 * W), m = q / (kFewN / 4), n = q % (kFewN / 4) * 4;
    if (q >= kQuads || m >= rows) continue;
    const float* part = f.part + (int64_t)tile * f.splits * kFewM * kFewN;
    f32x4 y = {};
    for (int sp = 0; sp < f.splits; sp += 8) {   // eight parts' loads in flight, added in order
      f32x4 v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = get_quad(part + (int64_t)min(sp + u, f.splits - 1) * kFewM * kFewN, kQuads, q);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (sp + u < f.splits) y += v[u];
    }
    finish(a, f.vec, m0 + m, n0 + n, y);
  }
}

// Slices of K a tile: as many as the chip has room for, of at least 16 chunks
// (64 x 1280 x 5120, 40 tiles: 1 / 2 / 4 / 5 / 6 / 10 slices 14.7 / 11.5 / 9.1 /
// 9.2 / 9.1 / 12 us; 64 x 1280 x 1280: 5.5 / 6.8 / 6.8).
int few_splits(const c4s_linear_desc& a, int64_t tiles) {
  const int chunks = (a.K + kChunk - 1) / kChunk;
  const int64_t most = chunks / 16, want = 256 / tiles;
  return (int)(want < 2 || most < 2 ? 1 : (want < most ? want : most));
}

template <bool Q8, int MB>
hipError_t few(const FewArgs& f, int64_t tiles, hipStream_t s) {
  const dim3 grid((unsigned)(tiles * f.splits));
  // Eight waves while every workgroup has a CU to itself (64 x 5120 x 1280, 160
  // workgroups: 6.7 us and 7.0; 1 x 3840 x 1280: 3.9 and 4.6), else four (200 x
  // 5120 x 1280, 640 workgroups: 15.7 us and 11.7).
  if (tiles * f.splits <= 256) hipLaunchKernelGGL((k_linear_few<Q8, MB, 8>), grid, dim3(512), 0, s, f);
  else hipLaunchKernelGGL((k_linear_few<Q8, MB, 4>), grid, dim3(256), 0, s, f);
  return hipGetLastError();
}

template <bool Q8>
hipError_t few(const FewArgs& f, int64_t tiles, hipStream_t s) {
  if (f.d.M <= 16) return few<Q8, 1>(f, tiles, s);
  if (f.d.M <= 32) return few<Q8, 2>(f, tiles, s);
  return few<Q8, 4>(f, tiles, s);
}

// ---- many rows --------------------------------------------------------------------------
//
// Tiles of outputs and rows, WN x WM waves of NW x MW fragments each.
struct ManyArgs {
  c4s_linear_desc d;
  bool vec;
  int m_tiles, n_tiles;
};

// The tile (outputs, rows) of this workgroup, in tiles; false if it has none.
// Workgroups go round the eight XCDs: each XCD gets a run of tiles of its own,
// eight tiles of rows by all outputs at a time, so that its L2 serves them.
__device__ __forceinline__ bool tile_of(const ManyArgs& f, int& n, int& m) {
  const int tiles = f.m_tiles * f.n_tiles, per = (tiles + 7) / 8;
  const int id = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
  if (id >= tiles || (int)(blockIdx.x / 8) >= per) return false;
  const int band = id / (8 * f.n_tiles), in = id % (8 * f.n_tiles);
  const int height = min(8, f.m_tiles - 8 * band);
  m = 8 * band + in % height;
  n = in / height;
  return true;
}

// Of the quads that lane group g (of the four of 16 lanes) has, q[i] number 4 i + g
// of a row, to q[2 s + e] number 8 s + 2 g + e: two pairs of quads next to each other.
__device__ __forceinline__ void swap_groups(uint32_t (&q)[4][2]) {
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const auto r = __builtin_amdgcn_permlane32_swap(q[i][e], q[i + 1][e], false, false);
      const auto t = __builtin_amdgcn_permlane16_swap(r[0], r[1], false, false);
      q[i][e] = t[0];
      q[i + 1][e] = t[1];
    }
}

// A wave's 4 x MW fragments from (m, n) on: lane (g, c) has outputs n + 16 i + 4 g ..
// + 3 of rows m + 16 j + c. Bias, activation and residual are applied as they lie;
// results in bf16 change lanes so that a store is of 32 outputs of a row next to each
// other.
// Stores go past the caches, which keeps the operands of the tiles in them (12345 x
// 5120 x 1280, gelu: 170 us, and 166 so; through LDS, a quad a lane: 170).
template <int MW>
__device__ __forceinline__ void write_tile(const ManyArgs& f, int m, int n, const f32x4 (&acc)[4][MW]) {
  const c4s_linear_desc& a = f.d;
  const int lane = threadIdx.x % 64, c = lane % 16, g = lane / 16;
  if (!f.vec) {
#pragma unroll
    for (int j = 0; j < MW; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (m + 16 * j + c < a.M) finish(a, false, m + 16 * j + c, n + 16 * i + 4 * g, acc[i][j]);
    return;
  }
  f32x4 b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = n + 16 * i + 4 * g;
    b[i] = a.bias && at < a.N ? *reinterpret_cast<const f32x4*>(a.bias + at) : f32x4{};
  }
#pragma unroll
  for (int j = 0; j < MW; ++j) {
    const int row = m + 16 * j + c;
    const bool in = row < a.M;
    f32x4 r[4] = {};
    if (a.residual && in) {
      const int64_t o = (int64_t)row * a.ld_res + n + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + 16 * i + 4 * g < a.N) r[i] = residual4(a, o + 16 * i);
    }
    float y[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = acc[i / 4][j][i % 4] + b[i / 4][i % 4];
    activate(y, a.act);
    if (a.residual) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] += r[i / 4][i % 4];
    }
    if (a.out_dtype == C4S_DTYPE_BF16) {
      uint32_t q[4][2];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i / 2][i % 2] = __builtin_bit_cast(uint32_t, Pair{(__bf16)y[2 * i], (__bf16)y[2 * i + 1]});
      swap_groups(q);
      uint16_t* o = static_cast<uint16_t*>(a.out) + (int64_t)row * a.ld_out + n + 8 * g;
#pragma unroll
      for (int i = 0; i < 4; i += 2, o += 32) {
        const int at = n + 16 * i + 8 * g;
        if (in && at + 8 <= a.N) __builtin_nontemporal_store(Eight{q[i][0], q[i][1], q[i + 1][0], q[i + 1][1]}, reinterpret_cast<Eight*>(o));
        else if (in && at < a.N) __builtin_nontemporal_store(u32x2{q[i][0], q[i][1]}, reinterpret_cast<u32x2*>(o));
      }
    } else if (in) {
      float* o = static_cast<float*>(a.out) + (int64_t)row * a.ld_out + n + 4 * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + 16 * i + 4 * g < a.N)
          __builtin_nontemporal_store(f32x4{y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]}, reinterpret_cast<f32x4*>(o + 16 * i));
    }
  }
}

// bf16. K in stages of 64 inputs, whose rows (128 bytes, in the permuted order of
// piece()) go from memory into LDS past the registers, two buffers. A wave's
// fragments are double buffered in registers too: while one half of a stage is
// multiplied, the next half's are read, so that the matrix engine waits only for
// the other waves at the barrier, once a stage. Eight waves on 256 x 256 reach
// 1330 TFLOP/s at 8192 x 8192 x 8192 (1265 when the others were tried: the rows in
// registers on the way and two barriers a stage 1030; stages of 32 inputs, four
// buffers 1190; 128 x 128 and two workgroups a CU 1060).
template <int NW, int MW, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM, WN * WM == 8 ? 1 : 2) void k_linear_many(ManyArgs f) {
  constexpr int kN = 16 * NW * WN, kM = 16 * MW * WM, kWaves = WN * WM, kStage = (kN + kM) * 128;
  constexpr int kLoads = (kN + kM) / 8 / kWaves;   // a wave's of a stage
  __shared__ __align__(128) char lds[2 * kStage];
  const c4s_linear_desc& a = f.d;
  const int t = threadIdx.x, lane = t % 64, wave = __builtin_amdgcn_readfirstlane(t / 64), c = lane % 16, g = lane / 16;
  int n0, m0;
  if (!tile_of(f, n0, m0)) return;
  n0 *= kN;
  m0 *= kM;
  const uint32_t xp = 2u * (uint32_t)a.ldx, wp = 2u * (uint32_t)a.K;
  const Tile xt(a.x + (int64_t)m0 * a.ldx, min(a.M - m0, kM), wp, xp);
  const Tile wt(static_cast<const uint16_t*>(a.weight) + (int64_t)n0 * a.K, min(a.N - n0, kN), wp, wp);
  // instruction j of the wave: rows r .. r + 7, r = 8 (kLoads wave + j); lane l row l / 8, and of it the piece that
  // piece() keeps at l % 8
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  const int stages = (a.K + 63) / 64;
  auto fetch = [&](int st) {
    const uint32_t dst = base + (uint32_t)(st % 2 * kStage) + 1024u * kLoads * wave;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int r = 8 * (kLoads * wave + j);
      const bool isx = r < kM;
      const uint32_t at = 16 * ((lane % 8) ^ (((r + lane / 8) >> 1) & 7));
      const bool in = (uint32_t)(st * 128) + at < wp;   // behind the last input: past the buffers' ends, where loads give zeros
      const uint32_t v = (isx ? (r + lane / 8) * xp : (r - kM + lane / 8) * wp) + at;
      // (m0, which says where in LDS, is the compiler's and cannot be named as clobbered: it is left as it was)
      uint32_t m0_was;
      asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                   : "=&s"(m0_was) : "s"(dst + 1024u * j), "v"(in ? v + 128u * st : 0x80000000u), "s"(isx ? xt.d : wt.d) : "memory");
    }
  };
  const int wn = wave % WN * 16 * NW, wm = wave / WN * 16 * MW;
  f32x4 acc[NW][MW] = {};
  struct Frags { uint4 w[NW], x[MW]; };
  auto read = [&](Frags& f, int st, int h) {
    const int o = st % 2 * kStage + piece(c, 4 * h + g);
#pragma unroll
    for (int i = 0; i < NW; ++i) f.w[i] = *reinterpret_cast<const uint4*>(lds + o + (kM + wn) * 128 + 2048 * i);
#pragma unroll
    for (int j = 0; j < MW; ++j) f.x[j] = *reinterpret_cast<const uint4*>(lds + o + wm * 128 + 2048 * j);
  };
  auto mul = [&](const Frags& f) {
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < MW; ++j)
#pragma unroll
      for (int i = 0; i < NW; ++i) acc[i][j] = mfma(f.w[i], f.x[j], acc[i][j]);
    __builtin_amdgcn_sched_barrier(0);
  };
  fetch(0);
  fetch(1);   // behind the last input: zeros
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(kLoads) : "memory");
  Frags fa, fb;
  read(fa, 0, 0);
  for (int st = 0; st < stages; ++st) {
    read(fb, st, 1);
    mul(fa);
    // every wave's rows of the next stage are there, and this stage's have been read by all
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    read(fa, st + 1, 0);
    fetch(st + 2);
    mul(fb);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // nothing on its way into LDS any more
  write_tile(f, m0 + wm, n0 + wn, acc);
}

// 8-bit codes: 128 x 128, four waves, two workgroups a CU. The codes pass through
// registers on their way into LDS, where they become q - 128; a chunk's products
// are scaled and added to the sums in fp32, as with few rows. 12345 x 5120 x 1280, group
// 64: 325 us, 500 TFLOP/s (bf16 weights: 165). One buffer and two barriers a chunk, between
// which nothing is multiplied; VALU 58 % busy with conversion and scaling, matrix engine 26 %,
// a fifth of that the sums of x, LDS 32 %.
__global__ __launch_bounds__(256, 2) void k_linear_many_q8(ManyArgs f) {
  constexpr int NW = 4, MW = 4, WN = 2, WM = 2, kN = 16 * NW * WN, kM = 16 * MW * WM;
  constexpr int kXLoads = kM / 32, kWLoads = kN / 64;
  __shared__ __align__(16) char xs[(kM + kN) * 128];
  char* ws = xs + kM * 128;
  __shared__ __align__(16) float sc[2][2 * kN];   // [half of the chunk][scales, offsets]
  const c4s_linear_desc& a = f.d;
  const int t = threadIdx.x, lane = t % 64, wave = t / 64, c = lane % 16, g = lane / 16;
  int n0, m0;
  if (!tile_of(f, n0, m0)) return;
  n0 *= kN;
  m0 *= kM;
  const uint32_t xp = 2u * (uint32_t)a.ldx, wp = (uint32_t)a.K;   // rows apart
  const Tile xt(a.x + (int64_t)m0 * a.ldx, min(a.M - m0, kM), 2u * a.K, xp);
  const Tile wt(static_cast<const char*>(a.weight) + (int64_t)n0 * wp, min(a.N - n0, kN), wp, wp);
  const uint32_t xo = t / 8 * xp + t % 8 * 16, wo = t / 4 * wp + t % 4 * 16;
  uint4 xv[kXLoads], wv[kWLoads];
  float sv[2];
  static_assert(2 * kN == 256, "a scale or offset a thread");
  const float* sr = (t < kN ? a.wscale : a.wbias) + (int64_t)min(n0 + t % kN, a.N - 1) * (a.K / a.group);
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < kXLoads; ++j) xv[j] = xt.load(xo + 32 * j * xp + 2 * k0);
#pragma unroll
    for (int j = 0; j < kWLoads; ++j) {   // codes are aligned to 8 bytes
      const uint2 lo = wt.load8(wo + 64 * j * wp + k0), hi = wt.load8(wo + 64 * j * wp + k0 + 8);
      wv[j] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
    const int gi = k0 / a.group;
    sv[0] = sr[gi];
    sv[1] = a.group == 32 ? sr[min(gi + 1, a.K / 32 - 1)] : sv[0];
  };
  auto stage = [&](int k0) {
    if (k0 + kChunk > a.K && k0 + t % 8 * 8 >= a.K) {   // inputs behind the last (codes are finite whatever they are)
#pragma unroll
      for (int j = 0; j < kXLoads; ++j) xv[j] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < kXLoads; ++j) *reinterpret_cast<uint4*>(xs + piece(t / 8 + 32 * j, t % 8)) = xv[j];
#pragma unroll
    for (int j = 0; j < kWLoads; ++j) {
      *reinterpret_cast<uint4*>(ws + piece(t / 4 + 64 * j, t % 4 * 2)) = centred(make_uint2(wv[j].x, wv[j].y));
      *reinterpret_cast<uint4*>(ws + piece(t / 4 + 64 * j, t % 4 * 2 + 1)) = centred(make_uint2(wv[j].z, wv[j].w));
    }
    sc[0][t] = sv[0];
    sc[1][t] = sv[1];
  };
  const int wn = wave % WN * 16 * NW, wm = wave / WN * 16 * MW;
  f32x4 acc[NW][MW] = {};
  load(0);
  for (int k0 = 0; k0 < a.K; k0 += kChunk) {
    if (k0) __syncthreads();   // the chunk before has been read
    stage(k0);
    __syncthreads();
    if (k0 + kChunk < a.K) load(k0 + kChunk);
    f32x4 part[NW][MW] = {}, sum[MW] = {};
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      uint4 x[MW];
      const uint32_t one = 0x3F803F80u;
#pragma unroll
      for (int j = 0; j < MW; ++j) {
        x[j] = *reinterpret_cast<const uint4*>(xs + piece(wm + 16 * j + c, 4 * st + g));
        sum[j] = mfma(make_uint4(one, one, one, one), x[j], sum[j]);
      }
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(ws + piece(wn + 16 * i + c, 4 * st + g));
#pragma unroll
        for (int j = 0; j < MW; ++j) part[i][j] = mfma(w, x[j], part[i][j]);
      }
      if (st == 0 && a.group != 32) continue;
#pragma unroll
      for (int i = 0; i < NW; ++i) {
        const f32x4 s = *reinterpret_cast<const f32x4*>(&sc[st][wn + 16 * i + 4 * g]), o = *reinterpret_cast<const f32x4*>(&sc[st][kN + wn + 16 * i + 4 * g]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float off = __builtin_fmaf(128.0f, s[e], o[e]);
#pragma unroll
          for (int j = 0; j < MW; ++j) {
            acc[i][j][e] = __builtin_fmaf(s[e], part[i][j][e], __builtin_fmaf(off, sum[j][e], acc[i][j][e]));
            part[i][j][e] = 0.0f;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < MW; ++j) sum[j] = f32x4{};
    }
  }
  write_tile(f, m0 + wm, n0 + wn, acc);
}

template <int NW, int MW, int WN, int WM>
ManyArgs many_args(const c4s_linear_desc& a) {
  constexpr int kN = 16 * NW * WN, kM = 16 * MW * WM;
  return ManyArgs{a, vectors(a), (a.M + kM - 1) / kM, (a.N + kN - 1) / kN};
}
dim3 many_grid(const ManyArgs& f) { return dim3((unsigned)(((int64_t)f.m_tiles * f.n_tiles + 7) / 8 * 8)); }

int64_t tiles_of(const c4s_linear_desc& a, int m, int n) {
  return (int64_t)((a.M + m - 1) / m) * ((a.N + n - 1) / n);
}

// Which kernel. Few rows' tiles (32 outputs by 64 rows) cost about alike, and
// from 1280 of them on the others win (us, bf16, K = 1280, N = 5120: 512 rows 19
// and 21, 640 rows 23 and 21, 1024 rows 31 and 24; K = 5120, N = 1280: 2000 rows 59
// and 59; 8-bit, N = 5120: 512 rows 31 and 39, 800 rows 46 and 45).
// With outputs so many that a single tile of rows exceeds that, the others' tiles are mostly rows
// that are not there. 8-bit codes cost them their conversion all the same, so up to 64 rows stay here (N = 151936,
// few / many, us: K = 1280: 1 row 58 / 110, 16 68 / 111, 64 107 / 116; K = 4096: 221 / 341, 247 / 344, 324 / 352). With
// bf16, weights are all that counts: here as far as x is small beside them, and while rows are not 8 KB apart
// or more, which whole stages take better (1 row: N = 151936, K = 1280 64 / 82, 3200 168 / 188, 4096 234 / 235; N =
// 70000, K = 2560 61 / 95; 16 rows: 76 / 84, 183 / 189, 255 / 238; 71 / 97; 48 rows: 97 / 95, 231 / 196).
bool few_pays(const c4s_linear_desc& a) {
  if (a.wdtype == C4S_W_Q8) return a.M <= kFewM || tiles_of(a, kFewM, kFewN) <= 1600;
  return (a.M <= 16 && a.K < 4096) || tiles_of(a, kFewM, kFewN) <= 1280;
}

// 128 x 128, two workgroups a CU, or 256 x 256: a round of the chip with the former
// takes 9/16 of one with the latter, which does twice the work (128 / 256, us: 1600 x
// 5120 x 1280, 2 and 1 rounds, 43 / 40; 4096, 3 and 2, 67 / 78; 5000, 4 and 2, 88 / 78;
// 7000, 5 and 3, 111 / 117; 12345, 8 and 4, 188 / 160; 4000 x 1280 x 1280, one, 24 / 39).
bool small_tiles_pay(const c4s_linear_desc& a) {
  const int64_t small = (tiles_of(a, 128, 128) + 511) / 512, large = (tiles_of(a, 256, 256) + 255) / 256;
  return 9 * small <= 16 * large;
}

}  // namespace

LayerSpace linear_space(const c4s_linear_desc& a) {
  if (!few_pays(a)) return {};
  const int64_t tiles = tiles_of(a, kFewM, kFewN);
  const int splits = few_splits(a, tiles);
  if (splits == 1) return {};
  return {tiles, tiles * splits * kFewM * kFewN};
}

hipError_t launch_linear(const c4s_linear_desc& a, uint32_t* counters, float* space, hipStream_t s) {
  if (few_pays(a)) {
    const int64_t tiles = tiles_of(a, kFewM, kFewN);
    const FewArgs f{a, vectors(a), few_splits(a, tiles), (a.N + kFewN - 1) / kFewN, counters, space};
    return a.wdtype == C4S_W_Q8 ? few<true>(f, tiles, s) : few<false>(f, tiles, s);
  }
  if (a.wdtype == C4S_W_Q8) {
    const ManyArgs f = many_args<4, 4, 2, 2>(a);
    hipLaunchKernelGGL(k_linear_many_q8, many_grid(f), dim3(256), 0, s, f);
  } else if (small_tiles_pay(a)) {
    const ManyArgs f = many_args<4, 4, 2, 2>(a);
    hipLaunchKernelGGL((k_linear_many<4, 4, 2, 2>), many_grid(f), dim3(256), 0, s, f);
  } else {
    const ManyArgs f = many_args<4, 8, 4, 2>(a);
    hipLaunchKernelGGL((k_linear_many<4, 8, 4, 2>), many_grid(f), dim3(512), 0, s, f);
  }
  return hipGetLastError();
}

}  // namespace c4s
