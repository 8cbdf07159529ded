// Rotary positions (c4s_rope, include/c4s_batch.h).
//
// A workgroup has one row, or a part of its heads: its first threads turn the
// position into cosines and sines, once for all heads, and leave them in LDS
// while every thread's first pieces of queries or keys are on their way. A piece is
// eight bf16 or four floats (of either half of the pairs, with C4S_ROPE_HALF), or
// single pairs where sizes or alignment do not allow that. Memory bounds it: stores go
// past the L2, where nothing would be found again (the next call's workgroups are on
// other dies). 18829 rows in place, halves, from the last-level cache, where the product
// before leaves them / from memory: 20 and 20 heads of 64 34 us, 5.6 TB/s / 45 (a half is
// half a line there); 32 and 8 of 128 59, 6.5 TB/s / 77. 20 and 20 heads of 64 in floats, of twice the bytes, 77 from memory, 5.0 TB/s.
// (Stores through the L2: 46 / 59 for heads of 64.
// Loads past the caches as well: 43 / 44, and 66 / 67 for heads of 128. One piece of a thread at a time 47 from memory;
// lines whole and the halves exchanged between lanes 48; workgroups of two or four rows 44.) 64 rows: 2.9 us.
//
// The angle is reduced in twice 64 bits: what the product position * frequency and its division by 2 pi (a
// constant of two parts) lose in their last place is added to what is left of the whole turns, of which there may be
// 2^28 and more. That rest, at most half a turn, is exact enough in 32 bits (2^-26 of a turn, 1e-7 radians). With 64 bits alone the
// error was more than 2^-52 of the number of turns: 3e-7 radians at frequency 1 and position 2^31, 3e-4 at
// frequency 1000. The calls take as long as before.

#include <hip/hip_runtime.h>

#include <algorithm>

#include "c4s_batch.hpp"

namespace c4s {
namespace {

constexpr int kRopePairs = 512;   // head_dim / 2 at most

// The sequence's position of packed row r; -1: it has none.
__device__ __forceinline__ int64_t position_of(const c4s_rope_desc& a, int r) {
  if (a.pos) return a.pos[r];
  int seq = r, left = 1;
  if (a.rows_off) {
    int lo = 0, hi = a.n_seqs;   // the last sequence that starts at or before r, eight parts a step
    while (hi - lo > 1) {
      const int step = (hi - lo + 7) / 8;
      int behind = 0;
#pragma unroll
      for (int j = 1; j < 8; ++j) behind += (lo + j * step < hi) & (a.rows_off[min(lo + j * step, hi - 1)] <= r);
      lo += behind * step;
      hi = min(lo + step, hi);
    }
    seq = lo;
    left = a.rows_off[seq + 1] - r;
    if (a.n_seqs == 0 || r < a.rows_off[seq] || left < 1) return -1;
  } else if (seq >= a.n_seqs) {
    return -1;
  }
  return max((int64_t)a.lens[seq] - left, (int64_t)-1);
}

typedef __bf16 bf16_t;
// N values of T, in memory that is aligned for them, or (one value or pair) for one.
template <class T, int N>
struct alignas(N <= 2 ? sizeof(T) : sizeof(T) * N) Few {
  T v[N];
};

// pos * freq / 2 pi less its whole turns.
__device__ __forceinline__ double part_of_turn(double pos, double freq) {
  constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnRest = -0x1.6b01ec5417056p-57;   // 1 / 2 pi
  const double angle = pos * freq, angle_rest = fma(pos, freq, -angle);
  const double turns = angle * kTurn;
  const double rest = fma(angle, kTurn, -turns) + (angle * kTurnRest + angle_rest * kTurn);
  return turns - rint(turns) + rest;
}

constexpr int kRopeThreads = 256, kRopeAhead = 2;   // pieces of a thread that are on their way together

typedef uint32_t Words __attribute__((ext_vector_type(4)));
template <class V>
__device__ __forceinline__ void put(V* to, const V& v) {
  if constexpr (sizeof(V) == 16) __builtin_nontemporal_store(__builtin_bit_cast(Words, v), reinterpret_cast<Words*>(to));
  else *to = v;
}

// Values of a piece that is not turned: single ones beside single pairs, as their number may be odd.
template <int N, bool PAIRS>
__host__ __device__ constexpr int copied() {
  return PAIRS && N == 2 ? 1 : N;
}

struct RopeArgs {
  c4s_rope_desc d;
  int parts;   // workgroups of a row
};

// T: of the tensors; N: values a piece; PAIRS: the layout.
template <class T, int N, bool PAIRS>
__global__ __launch_bounds__(kRopeThreads) void k_rope(RopeArgs f) {
  __shared__ float cs[kRopePairs], sn[kRopePairs];
  const c4s_rope_desc& a = f.d;
  const int row = blockIdx.x / f.parts, part = blockIdx.x % f.parts;
  const int half = a.rot_dim / 2;
  const int turned = (PAIRS ? a.rot_dim : half) / N;  // pieces of a head that are turned; the others
  constexpr int kCopy = copied<N, PAIRS>();
  const int per = turned + (a.head_dim - a.rot_dim) / kCopy;    // (copied) follow them
  const int heads = (a.q ? a.n_heads : 0) + (a.k ? a.n_kv_heads : 0), all = heads * per;
  const int step = blockDim.x * f.parts;

  struct Piece {
    const T* from;
    T* to;
    int at;    // its first value's place in the head; -1: copied
  };
  auto piece = [&](int i) {
    const int head = i / per, p = i - head * per;
    const bool is_q = a.q && head < a.n_heads;
    const int h = is_q || !a.q ? head : head - a.n_heads;
    const int64_t r = row;
    const T* from = static_cast<const T*>(is_q ? a.q : a.k) + r * (is_q ? a.ldq : a.ldk) + (int64_t)h * a.head_dim;
    T* to = static_cast<T*>(is_q ? a.q_out : a.k_out) + r * (is_q ? a.ldq_out : a.ldk_out) + (int64_t)h * a.head_dim;
    const int at = p < turned ? p * N : a.rot_dim + (p - turned) * kCopy;
    return Piece{from + at, to + at, p < turned ? at : -1};
  };
  using V = Few<T, N>;
  Piece now[kRopeAhead];
  V x[kRopeAhead], y[kRopeAhead];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kRopeAhead; ++u) {
      const int i = i0 + u * step;
      if (i >= all) continue;
      now[u] = piece(i);
      if (kCopy == N || now[u].at >= 0) x[u] = *reinterpret_cast<const V*>(now[u].from);
      else x[u].v[0] = *now[u].from;
      if (!PAIRS && now[u].at >= 0) y[u] = *reinterpret_cast<const V*>(now[u].from + half);
    }
  };
  int i = part * blockDim.x + threadIdx.x;
  load(i);

  const int64_t pos = position_of(a, row);
  if (pos < 0) return;
  for (int p = threadIdx.x; p < half; p += blockDim.x) {
    float s, c;
    sincospif(2.0f * (float)part_of_turn((double)pos, a.freq[p]), &s, &c);
    cs[p] = c * a.scale;
    sn[p] = s * a.scale;
  }
  __syncthreads();
  while (i < all) {
#pragma unroll
    for (int u = 0; u < kRopeAhead; ++u) {
      if (i + u * step >= all) continue;
      const int at = now[u].at;
      T* const to = now[u].to;
      V o;
      if (at < 0) {
        if (to == now[u].from) continue;
        if (kCopy == N) put(reinterpret_cast<V*>(to), x[u]);
        else *to = x[u].v[0];
      } else if constexpr (PAIRS) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float c = cs[(at + j) / 2], s = sn[(at + j) / 2], v = (float)x[u].v[j], w = (float)x[u].v[j + 1];
          o.v[j] = (T)(v * c - w * s);
          o.v[j + 1] = (T)(v * s + w * c);
        }
        put(reinterpret_cast<V*>(to), o);
      } else {
        V e;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const float c = cs[at + j], s = sn[at + j], v = (float)x[u].v[j], w = (float)y[u].v[j];
          o.v[j] = (T)(v * c - w * s);
          e.v[j] = (T)(v * s + w * c);
        }
        put(reinterpret_cast<V*>(to), o);
        put(reinterpret_cast<V*>(to + half), e);
      }
    }
    i += kRopeAhead * step;
    load(i);
  }
}

template <class T, int N, bool PAIRS>
hipError_t rope(const c4s_rope_desc& a, hipStream_t s) {
  const int per = (PAIRS ? a.rot_dim : a.rot_dim / 2) / N + (a.head_dim - a.rot_dim) / copied<N, PAIRS>();
  const int64_t all = (int64_t)((a.q ? a.n_heads : 0) + (a.k ? a.n_kv_heads : 0)) * per;
  // few rows: every thread has one piece; rows that fill the chip: kRopeAhead, in as many even rounds as that takes
  int parts = 1;
  int64_t threads = std::min<int64_t>(all, kRopeThreads);
  if (a.n_rows < 1024) {
    parts = (int)std::min<int64_t>((all + kRopeThreads - 1) / kRopeThreads, std::max(2048 / a.n_rows, 1));
  } else {
    const int64_t rounds = (all + kRopeAhead * kRopeThreads - 1) / (kRopeAhead * kRopeThreads);
    threads = (all + rounds * kRopeAhead - 1) / (rounds * kRopeAhead);
  }
  hipLaunchKernelGGL((k_rope<T, N, PAIRS>), dim3((unsigned)(a.n_rows * parts)), dim3((unsigned)((threads + 63) / 64 * 64)), 0, s, RopeArgs{a, parts});
  return hipGetLastError();
}

// Whether every piece of N values starts on its own size: sizes, strides, addresses.
bool fits(const c4s_rope_desc& a, int n, int size) {
  uint64_t odd = (uint64_t)a.head_dim | (uint64_t)(a.layout == C4S_ROPE_PAIRS ? a.rot_dim : a.rot_dim / 2) | (uint64_t)(a.head_dim - a.rot_dim);
  uint64_t at = 0;
  if (a.q) odd |= (uint64_t)(a.ldq | a.ldq_out), at |= (uint64_t)(uintptr_t)a.q | (uint64_t)(uintptr_t)a.q_out;
  if (a.k) odd |= (uint64_t)(a.ldk | a.ldk_out), at |= (uint64_t)(uintptr_t)a.k | (uint64_t)(uintptr_t)a.k_out;
  return odd % n == 0 && at % (n * size) == 0;
}

template <class T, int N>
hipError_t by_layout(const c4s_rope_desc& a, hipStream_t s) {
  const bool wide = fits(a, N, sizeof(T));
  if (a.layout == C4S_ROPE_HALF) return wide ? rope<T, N, false>(a, s) : rope<T, 1, false>(a, s);
  return wide ? rope<T, N, true>(a, s) : rope<T, 2, true>(a, s);
}

}  // namespace

hipError_t launch_rope(const c4s_rope_desc& a, hipStream_t s) {
  return a.dtype == C4S_DTYPE_BF16 ? by_layout<bf16_t, 8>(a, s) : by_layout<float, 4>(a, s);
}

}  // namespace c4s
